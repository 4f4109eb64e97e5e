"""Layer norm, linear attention with a decay per head and attention with a sliding window and sinks, on the GPU, against
their float64 forms (oracle/sequence_ref.py).

Tolerances, derived before the first run.  u = half a step of the element type (bf16 2^-8; float32 products and sums are
counted in 2^-24).  An output is rounded once: u |ref|.  Inside, bfloat16 kernels round the weights (and the copy of the
state that q meets) once, each error at most u of its term, so at most u `mag`, mag being the sum of the terms' absolute
values; the softmax's dS carries two (the weight itself, and rowsum(dO O) formed from the rounded o).  A float32 sum of n
terms is off by at most n 2^-24 mag.  A softmax weight inherits the absolute error of its score, (dim + 4) 2^-24 `size`, once
from itself and once from the sum it is divided by; powers of the decay are exponentials of at most 87 (larger ones vanish):
90 2^-24."""
import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from oracle import sequence_ref as ref

pytestmark = pytest.mark.gpu

U = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}
ULP = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def _rand(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen, device='cuda') * scale).to(dtype)


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _close(got, want, mag, inner, dtype, what):
    """|got - want| <= inner * mag + (u + 2^-24) |want|, elementwise; NaN nowhere."""
    err = (got.double() - want).abs()
    tol = inner * mag + (U[dtype] + ULP) * want.abs() + 1e-38
    worst = float((err / tol).max()) if err.numel() else 0.0
    assert worst <= 1.0, '%s: %.2f of the tolerance' % (what, worst)


# ---- layer norm ----

@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,cols', [(1, 1), (3, 2), (1, 7), (1000, 24), (333, 30), (65, 64), (2048, 900), (5, 1025), (700, 1024), (17, 2047),
                                       (9, 4096), (3, 16384), (4, 20001), (2, 40000)])
def test_layer_norm(vad, dtype, rows, cols):
    g = _gen(rows * 7 + cols)
    x = (_rand(g, rows, cols) * 2 + 3).to(dtype).requires_grad_()
    w = (1 + _rand(g, cols, scale=0.3)).requires_grad_()
    b = _rand(g, cols).requires_grad_()
    dy = _rand(g, rows, cols, dtype=dtype)
    y = vad.layer_norm(x, w, b)
    assert y.dtype == dtype and y.shape == x.shape
    grads = torch.autograd.grad(y, (x, w, b), dy)
    want = ref.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    xd = x.detach().double()
    r = 1 / torch.sqrt(xd.var(1, unbiased=False, keepdim=True) + 1e-5)
    # a row's sum: at most 160 values down a lane (256 lanes, 40000 columns) and 9 levels across; one deviation from the mean
    # is off by that of the largest value, then a few roundings
    n = 180 * ULP
    xh = ((xd - xd.mean(1, keepdim=True)) * r).abs()
    size = xd.abs().amax(1, keepdim=True) * r                     # what an error of the mean, relative to x, does to xh
    mag_xh = size + xh * (1 + size * size)                        # and through the variance
    _close(y.detach(), want[0], mag_xh * w.detach().abs() + b.detach().abs(), n, dtype, 'y')
    gw = (dy.double() * w.detach()).abs()
    mag = r * (gw + gw.mean(1, keepdim=True) + (xh + mag_xh) * (gw * (xh + mag_xh)).mean(1, keepdim=True)) * (1 + size * size)
    _close(grads[0], want[1], mag, n, dtype, 'dx')
    rows_n = (rows + 64) * ULP
    _close(grads[1], want[2], (dy.double().abs() * (xh + mag_xh)).sum(0), rows_n + n, torch.float32, 'dw')
    _close(grads[2], want[3], dy.double().abs().sum(0), rows_n, torch.float32, 'db')


@pytest.mark.parametrize('dtype', DTYPES)
def test_layer_norm_of_two_columns(vad, dtype):
    """dx is what eps leaves of g, a millionth here: right to a few roundings of g, not of g less its projection.  Four or so
    on the way to 1 / sqrt(var + eps), three times over, and four more; x - mean is exact to 2 ulp of x."""
    g = _gen(7)
    x = (_rand(g, 100, 2) * 2 + 0.5)
    x[0] = 1.0                                              # no variance: all of g - mean g
    x = x.to(dtype).requires_grad_()
    w = (1 + _rand(g, 2, scale=0.3))
    dy = _rand(g, 100, 2, dtype=dtype)
    for view in (x, x[:, [1, 0]], torch.cat((x, x), 1)[:, 1:3]):           # the last: rows that end inside a word
        dx = torch.autograd.grad(vad.layer_norm(view, w), view, dy)[0]
        want = ref.layer_norm(view.detach(), w, None, 1e-5, dy)[1]
        xd = view.detach().double()
        r = 1 / torch.sqrt(xd.var(1, unbiased=False, keepdim=True) + 1e-5)
        mag = 1e-5 * r ** 3 * (dy.double() * w).abs().sum(1, keepdim=True) * (1 + (xd.abs().amax(1, keepdim=True) * r) ** 2)
        _close(dx, want, mag.expand_as(xd), 30 * ULP, dtype, 'dx')


def test_layer_norm_parameters_shapes_and_strides(vad):
    g = _gen(5)
    x = _rand(g, 4, 6, 48)
    w16, b16 = (1 + _rand(g, 48)).bfloat16(), _rand(g, 48).bfloat16()
    plain = ref.layer_norm(x, None, None, 1e-5)
    assert float((vad.layer_norm(x).double() - plain).abs().max()) < 1e-5
    assert float((vad.layer_norm(x, bias=b16.float()).double() - plain - b16.double()).abs().max()) < 1e-5
    y16 = vad.layer_norm(x.bfloat16(), w16, b16)
    want = ref.layer_norm(x.bfloat16(), w16, b16, 1e-5)
    assert float(((y16.double() - want).abs() / (want.abs() + 1e-2)).max()) < 2.0 ** -8 + 1e-4
    # bfloat16 parameters get bfloat16 gradients
    leaf = [t.clone().requires_grad_() for t in (x.bfloat16(), w16, b16)]
    dy = _rand(g, 4, 6, 48, dtype=torch.bfloat16)
    grads = torch.autograd.grad(vad.layer_norm(*leaf), leaf, dy)
    exact = ref.layer_norm(leaf[0].detach(), w16, b16, 1e-5, dy)
    for got, e in zip(grads, exact[1:]):
        assert got.dtype == torch.bfloat16
        assert float(((got.double() - e).abs() / (e.abs() + 1e-2)).max()) < 2.0 ** -8 + 1e-3
    # only some of the gradients, and every stride: the same bits as dense rows
    wide = _rand(g, 40, 100)
    for view in (wide[:, 3:51], wide[::2, :48], wide[:, :48].T.contiguous().T, wide[:1, :48].expand(40, 48), wide[:, ::2]):
        leaf = view.detach().requires_grad_()
        w = torch.ones(view.size(1), device='cuda')
        y = vad.layer_norm(leaf, w)
        dense = view.contiguous().requires_grad_()
        yd = vad.layer_norm(dense, w)
        assert torch.allclose(y, yd, rtol=1e-6, atol=1e-6)
        ones = torch.ones((), device='cuda').expand(y.shape)
        assert torch.allclose(torch.autograd.grad(y, leaf, ones)[0], torch.autograd.grad(yd, dense, ones)[0], atol=1e-5)
    # no rows; a row with a NaN leaves the others alone; huge offsets keep their variance
    empty = torch.empty(0, 24, device='cuda', requires_grad=True)
    we = torch.ones(24, device='cuda', requires_grad=True)
    ge = torch.autograd.grad(vad.layer_norm(empty, we), (empty, we), torch.empty(0, 24, device='cuda'))
    assert ge[0].shape == (0, 24) and not ge[1].any()
    x = _rand(g, 64, 24)
    clean = vad.layer_norm(x)
    x[10, 3] = math.nan
    dirty = vad.layer_norm(x)
    assert dirty[10].isnan().all() and torch.equal(dirty[:10], clean[:10]) and torch.equal(dirty[11:], clean[11:])
    far = torch.arange(24, device='cuda').float().repeat(8, 1) + 2.0 ** 20
    assert float((vad.layer_norm(far).double() - ref.layer_norm(far, None, None, 1e-5)).abs().max()) < 1e-5


# ---- linear attention ----

def _decays(heads):
    # forgetting within 2, 4, ... rows, never, and at once
    vals = [math.log1p(-2.0 ** -(1 + i)) for i in range(8)] + [0.0, -200.0]
    return torch.tensor([vals[(3 * i + 2) % len(vals)] for i in range(heads)], device='cuda')


def _decay_reference(q, k, v, log_decay, scale, starts, state, do, dstate):
    """Results and magnitudes laid out as the operator lays them out."""
    a = log_decay.clamp(-87.0, 0.0).double().tolist()
    seqs = [ref.sequences(t.detach().double(), starts) for t in (q, k, v, do)]
    out = {n: [] for n in ('o', 'dq', 'dk', 'dv', 'state', 'dstate')}
    out.update({'mag_' + n: [] for n in list(out)})
    for s, (qs, ks, vs, gs) in enumerate(zip(*seqs)):
        heads = [ref.decay_sequence(qs[:, h], ks[:, h], vs[:, h], a[h], scale, None if state is None else state[s, h].detach().double(),
                                    gs[:, h], None if dstate is None else dstate[s, h].double()) for h in range(len(a))]
        for n in out:
            out[n].append(torch.stack([x[n] for x in heads], 0 if 'state' in n else 1))
    join = torch.stack if starts is None else torch.cat
    return {n: torch.stack(x) if 'state' in n else join(x) for n, x in out.items()}


DECAY_CASES = [   # lengths, heads, dim, packed
    ([1], 1, 1, False), ([1, 1, 1], 2, 30, False), ([64], 2, 64, False), ([65, 65], 3, 33, False), ([63], 1, 128, False), ([166] * 3, 3, 30, False),
    ([700], 2, 64, False), ([1500], 1, 128, False), ([0, 5, 0, 131, 64, 1], 2, 64, True), ([300, 1100, 0], 3, 30, True), ([900, 20], 1, 96, True),
    ([1300], 2, 16, True),
]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('lengths,heads,dim,packed', DECAY_CASES)
def test_linear_attention(vad, dtype, lengths, heads, dim, packed):
    g = _gen(sum(lengths) + dim)
    lead = (sum(lengths),) if packed else (len(lengths), lengths[0])
    starts = torch.tensor([0] + lengths, device='cuda').cumsum(0) if packed else None
    q, k, v, do = (_rand(g, *lead, heads, dim, dtype=dtype) for _ in range(4))
    state, dstate = (_rand(g, len(lengths), heads, dim, dim) for _ in range(2))
    log_decay, scale = _decays(heads), 0.3
    leaf = [t.requires_grad_() for t in (q, k, v, state)]
    o, last = vad.linear_attention(*leaf[:3], log_decay, scale=scale, state=leaf[3], starts=starts, max_len=max(lengths))
    assert o.dtype == dtype and o.shape == q.shape and last.dtype == torch.float32
    grads = torch.autograd.grad((o, last), leaf, (do, dstate))
    want = _decay_reference(q, k, v, log_decay, scale, starts, state, do, dstate)
    pieces = -(-max(lengths) // 64)
    n = (2 * dim + 2 * 64 + 4 * pieces + 100) * ULP
    for name, got in (('o', o.detach()), ('dq', grads[0]), ('dk', grads[1]), ('dv', grads[2])):
        _close(got, want[name], want['mag_' + name], U[dtype] + n, dtype, name)
    for name, got in (('state', last.detach()), ('dstate', grads[3])):        # the state is exact to float32 in either type
        _close(got, want[name], want['mag_' + name], n, torch.float32, name)
    # without a state, and only the state's gradient
    o2, last2 = vad.linear_attention(q.detach(), k.detach(), v.detach(), log_decay, scale=scale, starts=starts)
    want = _decay_reference(q, k, v, log_decay, scale, starts, None, do, None)
    _close(o2, want['o'], want['mag_o'], U[dtype] + n, dtype, 'o from zero')
    _close(last2, want['state'], want['mag_state'], n, torch.float32, 'state from zero')
    again = vad.linear_attention(q.detach(), k.detach(), v.detach(), log_decay, scale=scale, starts=starts)
    assert torch.equal(o2, again[0]) and torch.equal(last2, again[1])


def test_linear_attention_gradients_against_differences(vad):
    g = _gen(3)
    q, k, v = (_rand(g, 2, 150, 2, 30) for _ in range(3))
    state = _rand(g, 2, 2, 30, 30)
    wo, ws = _rand(g, 2, 150, 2, 30), _rand(g, 2, 2, 30, 30)
    log_decay = torch.tensor([-0.05, 0.0], device='cuda')

    def loss(*t):
        o, s = vad.linear_attention(*t[:3], log_decay, state=t[3])
        return (o.double() * wo).sum() + (s.double() * ws).sum()

    leaf = [t.requires_grad_() for t in (q, k, v, state)]
    grads = torch.autograd.grad(loss(*leaf), leaf)
    # the loss is linear in each input by itself: a central difference of any length is exact but for rounding
    for i, got in enumerate(grads):
        d = _rand(g, *leaf[i].shape)
        with torch.no_grad():
            moved = [[t + s * d if j == i else t for j, t in enumerate(leaf)] for s in (0.5, -0.5)]
            slope = float(loss(*moved[0]) - loss(*moved[1]))
        assert slope == pytest.approx(float((got.double() * d).sum()), rel=2e-4, abs=2e-2)


def test_linear_attention_step_goes_on_from_a_recording(vad):
    for dtype in DTYPES:
        for heads, dim in ((3, 30), (2, 64), (1, 1), (4, 128), (2, 33)):
            g = _gen(dim)
            q, k, v = (_rand(g, 5, 80, heads, dim, dtype=dtype) for _ in range(3))
            log_decay = _decays(heads)
            whole, last = vad.linear_attention(q, k, v, log_decay)
            _, state = vad.linear_attention(q[:, :70], k[:, :70], v[:, :70], log_decay)
            want = _decay_reference(q, k, v, log_decay, dim ** -0.5, None, None, q, None)
            for t in range(70, 80):
                o = vad.linear_attention_step(q[:, t], k[:, t], v[:, t], log_decay, state)
                _close(o, want['o'][:, t], want['mag_o'][:, t], (dim + 150) * ULP, dtype, 'step %d' % t)
            _close(state, want['state'], want['mag_state'], (dim + 250) * ULP, torch.float32, 'state')


@pytest.mark.parametrize('dtype', DTYPES)
def test_linear_attention_later_rows_do_not_reach_earlier_ones(vad, dtype):
    """Infinities and NaN from row 100 on leave rows 0 .. 99 as they were, and the gradients the other way round; other
    sequences and heads feel nothing."""
    g = _gen(9)
    q, k, v, do = (_rand(g, 2, 200, 2, 64, dtype=dtype) for _ in range(4))
    log_decay = _decays(2)
    clean = vad.linear_attention(q, k, v, log_decay)[0]
    for which in range(3):
        t = [x.clone() for x in (q, k, v)]
        t[which][0, 100:, 0] = math.nan if which else math.inf
        o = vad.linear_attention(*t, log_decay)[0]
        assert torch.isfinite(o[0, :100]).all() and torch.isfinite(o[1]).all() and torch.isfinite(o[0, :, 1]).all()
        assert torch.allclose(o[0, :100].float(), clean[0, :100].float(), rtol=2 * U[dtype] + 1e-4, atol=1e-3)
        assert torch.equal(o[1], clean[1])
    leaf = [x.clone().requires_grad_() for x in (q, k, v)]
    bad = do.clone()
    bad[0, :100, 0] = math.nan
    grads = torch.autograd.grad(vad.linear_attention(*leaf, log_decay)[0], leaf, bad)
    for x in grads[1:]:
        assert torch.isfinite(x[0, 100:]).all() and torch.isfinite(x[1]).all()
    assert torch.isfinite(grads[0][0, 100:]).all()


# ---- window attention ----

def _window_reference(q, k, v, window, sinks, scale, starts, do):
    heads, group = q.size(-2), q.size(-2) // k.size(-2)
    seqs = [ref.sequences(t.detach().double(), starts) for t in (q, k, v, do)]
    out = {n: [] for n in ('o', 'dq', 'dk', 'dv', 'mag_o', 'mag_dq', 'mag_dk', 'mag_dv')}
    size = 0.0
    for qs, ks, vs, gs in zip(*seqs):
        per = [ref.window_sequence(qs[:, h], ks[:, h // group], vs[:, h // group], window, sinks, scale, gs[:, h]) for h in range(heads)]
        size = max([size] + [x['size'] for x in per])
        for n in out:
            t = torch.stack([x[n] for x in per], 1)
            out[n].append(t.unflatten(1, (heads // group, group)).sum(2) if n[-2:] in ('dk', 'dv') else t)
    join = torch.stack if starts is None else torch.cat
    return {n: join(x) for n, x in out.items()}, size


WINDOW_CASES = [   # lengths, heads, kv heads, dim, window, sinks, packed
    ([1], 1, 1, 1, 1, 0, False), ([1, 1], 2, 1, 30, 5, 3, False), ([64], 2, 2, 64, 64, 0, False), ([65], 3, 3, 33, 1, 0, False),
    ([200], 2, 1, 64, 30, 0, False), ([200] * 2, 4, 2, 64, 17, 4, False), ([300], 2, 1, 128, 100, 64, False), ([700], 3, 3, 30, 30, 0, False),
    ([500], 2, 1, 16, 1, 1, False), ([450], 1, 1, 96, 1000, 7, False), ([0, 3, 129, 0, 65, 256, 1], 4, 2, 64, 63, 2, True),
    ([700, 40], 6, 2, 30, 129, 20, True), ([1200, 0], 2, 1, 128, 256, 33, True), ([1700], 4, 1, 64, 40, 5, True),
]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('lengths,heads,kv_heads,dim,window,sinks,packed', WINDOW_CASES)
def test_window_attention(vad, dtype, lengths, heads, kv_heads, dim, window, sinks, packed):
    g = _gen(sum(lengths) + dim + window)
    lead = (sum(lengths),) if packed else (len(lengths), lengths[0])
    starts = torch.tensor([0] + lengths, device='cuda').cumsum(0) if packed else None
    q, do = (_rand(g, *lead, heads, dim, dtype=dtype) for _ in range(2))
    k, v = (_rand(g, *lead, kv_heads, dim, dtype=dtype) for _ in range(2))
    scale = 1.5 * dim ** -0.5
    leaf = [t.requires_grad_() for t in (q, k, v)]
    o = vad.window_attention(*leaf, window, sinks, scale=scale, starts=starts, max_len=max(lengths))
    assert o.dtype == dtype and o.shape == q.shape
    grads = torch.autograd.grad(o, leaf, do)
    want, size = _window_reference(q, k, v, window, sinks, scale, starts, do)
    n = (2 * (dim + 8) * max(size, 1.0) + max(lengths) + dim) * ULP
    _close(o.detach(), want['o'], want['mag_o'], U[dtype] + n, dtype, 'o')
    _close(grads[2], want['dv'], want['mag_dv'], U[dtype] + n * (heads // kv_heads), dtype, 'dv')
    _close(grads[0], want['dq'], want['mag_dq'], 2 * U[dtype] + 2 * n, dtype, 'dq')
    _close(grads[1], want['dk'], want['mag_dk'], 2 * U[dtype] + 2 * n * (heads // kv_heads), dtype, 'dk')
    with torch.no_grad():
        assert torch.equal(vad.window_attention(q, k, v, window, sinks, scale=scale, starts=starts), o)
    grads2 = torch.autograd.grad(vad.window_attention(*leaf, window, sinks, scale=scale, starts=starts, max_len=max(lengths)), leaf, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, grads2))


@pytest.mark.parametrize('length,dim,window,sinks', [(200, 64, 2, 0), (200, 30, 4, 1), (150, 128, 3, 0), (300, 64, 100, 4), (300, 16, 300, 0)])
def test_window_attention_gradients_keep_bfloat16(vad, length, dim, window, sinks):
    """Each result takes two roundings to bfloat16 -- of the weights (P or dS), of itself -- and nothing else that counts.  A
    rounding is off by up to 2^-8, evenly spread: 2^-8 / sqrt(3) in the mean square, two of them sqrt(2 / 3) 2^-8."""
    g = _gen(91)
    q, k, v, do = (_rand(g, 1, length, 2, dim, dtype=torch.bfloat16) for _ in range(4))
    leaf = [t.requires_grad_() for t in (q, k, v)]
    o = vad.window_attention(*leaf, window, sinks)
    got = (o, *torch.autograd.grad(o, leaf, do))
    for h in range(2):
        exact = [t.detach()[0, :, h].double().requires_grad_() for t in (q, k, v)]
        want = ref.window_sequence(*exact, window, sinks, dim ** -0.5)['o']
        for a, b in zip(got, (want, *torch.autograd.grad(want, exact, do[0, :, h].double()))):
            assert float((a.detach()[0, :, h].double() - b.detach()).norm()) <= (2 / 3) ** 0.5 * 2.0 ** -8 * float(b.detach().norm())


def test_window_attention_gradients_against_differences(vad):
    g = _gen(4)
    q = _rand(g, 1, 150, 4, 30)
    k, v = (_rand(g, 1, 150, 2, 30) for _ in range(2))
    w = _rand(g, 1, 150, 4, 30)
    leaf = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad((vad.window_attention(*leaf, 20, 3).double() * w).sum(), leaf)
    for i, got in enumerate(grads):
        d = _rand(g, *leaf[i].shape)
        h = 2.0 ** -6
        with torch.no_grad():
            ends = [float((vad.window_attention(*[t + s * h * d if j == i else t for j, t in enumerate(leaf)], 20, 3).double() * w).sum())
                    for s in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * h)
        # the third derivative's h^2 / 6 and the rounding of the two sums over 2 h
        assert slope == pytest.approx(float((got.double() * d).sum()), rel=2e-3, abs=5e-2)


@pytest.mark.parametrize('dtype', DTYPES)
def test_window_attention_masked_rows_have_no_influence(vad, dtype):
    """Infinities and NaN in keys and values that a row does not see -- later ones and those its window has left -- leave it
    as it was; so do NaN queries and output gradients of rows that do not see a key, for that key's gradients."""
    g = _gen(8)
    window, sinks, n = 40, 4, 300
    q, do = (_rand(g, 1, n, 2, 64, dtype=dtype) for _ in range(2))
    k, v = (_rand(g, 1, n, 1, 64, dtype=dtype) for _ in range(2))
    clean = vad.window_attention(q, k, v, window, sinks)
    at = 130
    rows = torch.arange(n, device='cuda')
    blind = (rows < at) | (rows >= at + window)
    for which, value in ((0, math.nan), (1, math.nan), (1, math.inf)):
        t = [k.clone(), v.clone()]
        t[which][0, at] = value
        o = vad.window_attention(q, *t, window, sinks)
        assert torch.isfinite(o[0, blind]).all() and not torch.isfinite(o[0, ~blind]).all()
        assert torch.allclose(o[0, blind].float(), clean[0, blind].float(), rtol=2 * U[dtype] + 1e-4, atol=2 * U[dtype] + 1e-4)
    keys = rows
    unseen = (keys > at) | ((keys <= at - window) & (keys >= sinks))
    for which in range(2):
        t = [q.clone(), do.clone()]
        t[which][0, at, 0] = math.nan
        leaf = [x.requires_grad_() for x in (t[0], k.clone(), v.clone())]
        grads = torch.autograd.grad(vad.window_attention(*leaf, window, sinks), leaf, t[1])
        for x in grads[1:]:
            assert torch.isfinite(x[0, unseen]).all() and not torch.isfinite(x[0, ~unseen]).all()
        assert torch.isfinite(grads[0][0, rows != at]).all() and torch.isfinite(grads[0][0, :, 1]).all()


STEP_CASES = [(1, 1, 1, 1, 1, 0), (3, 4, 2, 64, 30, 0), (2, 6, 2, 30, 100, 3), (2, 8, 1, 128, 700, 64), (1, 5, 5, 33, 257, 1), (4, 16, 4, 96, 64, 2)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('batch,heads,kv_heads,dim,window,sinks', STEP_CASES)
def test_window_attention_step(vad, dtype, batch, heads, kv_heads, dim, window, sinks):
    """Caches full of NaN, filled by recordings shorter and longer than they hold, then steps: every output is that of the
    whole recording's row."""
    g = _gen(window + dim)
    slots = sinks + window
    for length in (0, 1, sinks + 1, slots - 1 if slots > 1 else 1, slots, 2 * slots + 3):
        total = length + 3
        q = _rand(g, batch, total, heads, dim, dtype=dtype)
        k, v = (_rand(g, batch, total, kv_heads, dim, dtype=dtype) for _ in range(2))
        ck, cv = (torch.full((batch, slots, kv_heads, dim), math.nan, dtype=dtype, device='cuda') for _ in range(2))
        pos = vad.window_cache_fill(k[:, :length], v[:, :length], ck, cv, window, sinks)
        assert pos.tolist() == [length] * batch
        want, size = _window_reference(q, k, v, window, sinks, dim ** -0.5, None, q)
        tol = (2 * (dim + 8) * max(size, 1.0) + slots + dim) * ULP
        for t in range(length, total):
            o = vad.window_attention_step(q[:, t], k[:, t], v[:, t], ck, cv, pos, window, sinks)
            _close(o, want['o'][:, t], want['mag_o'][:, t], tol, dtype, 'length %d row %d' % (length, t))
            slot = ref.window_slot(t, window, sinks)
            assert torch.equal(ck[:, slot], k[:, t]) and torch.equal(cv[:, slot], v[:, t])
            pos += 1


def test_window_step_rows_at_different_places(vad):
    g = _gen(2)
    window, sinks, dim = 50, 2, 64
    pos = torch.tensor([0, -1, 1, 51, 2 ** 33 + 5, -7, 60], device='cuda')
    b = pos.numel()
    q, k, v = _rand(g, b, 4, dim), _rand(g, b, 2, dim), _rand(g, b, 2, dim)
    ck, cv = _rand(g, b, 52, 2, dim), _rand(g, b, 52, 2, dim)
    before = ck.clone(), cv.clone()
    o = vad.window_attention_step(q, k, v, ck, cv, pos, window, sinks)
    for i, p in enumerate(pos.tolist()):
        if p < 0:
            assert not o[i].any() and torch.equal(ck[i], before[0][i]) and torch.equal(cv[i], before[1][i])
            continue
        kk, vv = before[0][i].clone(), before[1][i].clone()
        slot = ref.window_slot(p, window, sinks)
        kk[slot], vv[slot] = k[i], v[i]
        assert torch.equal(ck[i], kk) and torch.equal(cv[i], vv)
        n = min(p + 1, 52)
        for h in range(4):
            w = torch.softmax(kk[:n, h // 2].double() @ q[i, h].double() * dim ** -0.5, 0)
            assert float((o[i, h].double() - w @ vv[:n, h // 2].double()).abs().max()) < 1e-5


# ---- what all share ----

def _packed_views(t):
    """The same values at other strides: a slice of a wider tensor, heads first, and one element off alignment."""
    yield torch.cat([t, t, t], -2)[..., t.size(-2):2 * t.size(-2), :]
    yield t.transpose(-3, -2).contiguous().transpose(-3, -2)
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.flatten()
    yield flat[1:].view(t.shape)
    yield t.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.parametrize('dtype', DTYPES)
def test_strides_and_alignment(vad, dtype):
    g = _gen(6)
    q, k, v, do = (_rand(g, 2, 130, 2, 64, dtype=dtype) for _ in range(4))
    log_decay = _decays(2)

    def everything(q, k, v, do):
        leaf = [t.detach().requires_grad_() for t in (q, k, v)]
        o, s = vad.linear_attention(*leaf, log_decay)
        w = vad.window_attention(*leaf, 50, 2)
        return [o, s, w, *torch.autograd.grad(o, leaf, do), *torch.autograd.grad(w, leaf, do)]

    want = everything(q, k, v, do)
    for views in zip(*(_packed_views(t) for t in (q, k, v, do))):
        for a, b in zip(everything(*views), want):
            assert torch.equal(a, b)
    # an expanded gradient, as sum().backward() gives
    leaf = [t.clone().requires_grad_() for t in (q, k, v)]
    vad.window_attention(*leaf, 50, 2).sum().backward()
    ones = torch.autograd.grad(vad.window_attention(*leaf, 50, 2), leaf, torch.ones_like(q))
    assert all(torch.equal(a.grad, b) for a, b in zip(leaf, ones))
    # steps on slices of a fused projection
    x = _rand(g, 3, 3, 2, 64, dtype=dtype)
    state = _rand(g, 3, 2, 64, 64)
    a = vad.linear_attention_step(x[:, 0], x[:, 1], x[:, 2], log_decay, state.clone())
    b = vad.linear_attention_step(*[x[:, i].contiguous() for i in range(3)], log_decay, state.clone())
    assert torch.equal(a, b)
    cache = _rand(g, 3, 2, 20, 2, 64, dtype=dtype)
    pos = torch.tensor([3, 19, 100], device='cuda')
    a = vad.window_attention_step(x[:, 0], x[:, 1], x[:, 2], cache[:, 0], cache[:, 1], pos, 20)
    cc = cache.clone()
    b = vad.window_attention_step(*[x[:, i].contiguous() for i in range(3)], cc[:, 0].contiguous(), cc[:, 1].contiguous(), pos, 20)
    assert torch.equal(a, b)


def test_rows_of_no_sequence(vad):
    """Rows before the first and behind the last sequence: NaN there reaches nothing, outputs and gradients there are zero; a
    table that reaches outside is cut off."""
    g = _gen(7)
    n, lo, hi = 300, 17, 260
    q, k, v, do = (_rand(g, n, 2, 64) for _ in range(4))
    for t in (q, k, v, do):
        t[:lo] = math.nan
        t[hi:] = math.nan
    starts = torch.tensor([lo, 100, 100, hi], device='cuda')
    log_decay = _decays(2)
    inner = torch.tensor([0, 100 - lo, 100 - lo, hi - lo], device='cuda')
    for call in (lambda *t, s: vad.linear_attention(*t, log_decay, starts=s)[0], lambda *t, s: vad.window_attention(*t, 30, 4, starts=s, max_len=200)):
        leaf = [t.clone().requires_grad_() for t in (q, k, v)]
        o = call(*leaf, s=starts)
        cut = [t[lo:hi].clone().requires_grad_() for t in (q, k, v)]
        oc = call(*cut, s=inner)
        grads, grads_c = torch.autograd.grad(o, leaf, do), torch.autograd.grad(oc, cut, do[lo:hi])
        for a, b in zip((o, *grads), (oc, *grads_c)):
            assert torch.allclose(a[lo:hi], b, rtol=1e-4, atol=1e-4) and not a[:lo].any() and not a[hi:].any()
        o = call(*[t.nan_to_num() for t in (q, k, v)], s=torch.tensor([-5, 100, 10 ** 12], device='cuda'))
        assert torch.isfinite(o).all()
        none = call(q, k, v, s=torch.tensor([5], device='cuda'))
        assert not none.any()


def test_empty_calls(vad):
    for lead in ((0, 10), (3, 0)):
        q, k, v = (torch.empty(*lead, 2, 32, device='cuda', requires_grad=True) for _ in range(3))
        state = torch.randn(lead[0], 2, 32, 32, device='cuda', requires_grad=True)
        o, s = vad.linear_attention(q, k, v, _decays(2), state=state)
        assert o.shape == q.shape and torch.equal(s, state)
        ds = torch.randn_like(s)
        assert torch.equal(torch.autograd.grad(s, state, ds)[0], ds)
        w = vad.window_attention(q, k, v, 5)
        assert torch.autograd.grad(w, q, torch.empty_like(w))[0].shape == q.shape
    z = torch.empty(0, 2, 32, device='cuda')
    assert vad.linear_attention_step(z, z, z, _decays(2), torch.empty(0, 2, 32, 32, device='cuda')).shape == (0, 2, 32)
    c = torch.empty(0, 6, 2, 32, device='cuda')
    assert vad.window_attention_step(z, z, z, c, c.clone(), torch.empty(0, dtype=torch.int64, device='cuda'), 6).shape == (0, 2, 32)


def test_other_streams_and_graphs(vad):
    vad.init()
    g = _gen(11)
    x = _rand(g, 2, 400, 192, dtype=torch.bfloat16)
    w, b = torch.ones(192, device='cuda'), torch.zeros(192, device='cuda')
    log_decay = _decays(3)
    state, cache = _rand(g, 2, 3, 64, 64), _rand(g, 2, 2, 34, 3, 64, dtype=torch.bfloat16)
    pos = torch.tensor([5, 70], device='cuda')

    def forward():
        h = vad.layer_norm(x, w, b).view(2, 400, 3, 64)
        o, s = vad.linear_attention(h, h, h, log_decay)
        y = vad.window_attention(h, o, h, 30, 4)
        st = vad.linear_attention_step(h[:, 0], h[:, 1], h[:, 2], log_decay, s)
        ct = vad.window_attention_step(h[:, 0], h[:, 1], h[:, 2], cache[:, 0], cache[:, 1], pos, 30, 4)
        return o, s, y, st, ct

    want = [t.clone() for t in forward()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = forward()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, r) for p, r in zip(got, want))

    leaf = x.view(2, 400, 3, 64).clone().requires_grad_()

    def train():
        h = vad.layer_norm(leaf)
        o, _ = vad.linear_attention(h, h, h, log_decay)
        y = vad.window_attention(o, h, o, 30, 4)
        return torch.autograd.grad(y, leaf, leaf.detach())[0]

    want_grad = train().clone()
    with torch.cuda.stream(side):
        for _ in range(2):
            forward(), train()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                     # two graphs alive at once keep to their own scratch
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = forward(), train()
        graphs.append((graph, out))
    for turn in range(3):
        for graph, _ in graphs:
            graph.replay()
        (torch.randn(1000, device='cuda') * 2).sum().item()
        for graph, (out, grad) in graphs:
            assert all(torch.equal(p, r) for p, r in zip(out, want)) and torch.equal(grad, want_grad)
    torch.cuda.synchronize()


def test_gradient_of_the_state_alone(vad):
    g = _gen(21)
    q, k, v = (_rand(g, 2, 100, 2, 30).requires_grad_() for _ in range(3))
    state = _rand(g, 2, 2, 30, 30).requires_grad_()
    ds = _rand(g, 2, 2, 30, 30)
    log_decay = _decays(2)
    grads = torch.autograd.grad(vad.linear_attention(q, k, v, log_decay, state=state)[1], (q, k, v, state), ds)
    want = _decay_reference(q, k, v, log_decay, 30 ** -0.5, None, state, torch.zeros_like(q), ds)
    assert not grads[0].any()
    for got, name in zip(grads[1:], ('dk', 'dv', 'dstate')):
        _close(got, want[name], want['mag_' + name], 400 * ULP, torch.float32, name)


def test_offsets_past_32_bits(vad):
    """More than 2^31 elements in a tensor: the far end computes as a short call does."""
    n, heads, dim = 1_060_000, 16, 128
    g = _gen(31)
    x = torch.empty(n, heads, dim, dtype=torch.bfloat16, device='cuda')
    assert x.numel() > 2 ** 31
    x.zero_()
    tail = 300
    x[-tail:] = _rand(g, tail, heads, dim, dtype=torch.bfloat16)
    starts = torch.tensor([0, n - tail, n], device='cuda')
    short = x[-tail:].clone()
    inner = torch.tensor([0, tail], device='cuda')
    log_decay = _decays(heads)
    o, s = vad.linear_attention(x, x, x, log_decay, starts=starts, max_len=n)
    oc, sc = vad.linear_attention(short, short, short, log_decay, starts=inner)
    assert torch.allclose(o[-tail:].float(), oc.float(), rtol=2.0 ** -6, atol=1e-2) and torch.allclose(s[1], sc[0], rtol=1e-4, atol=1e-4)
    assert not o[:-tail].any()
    del o
    w = vad.window_attention(x, x, x, 50, 4, starts=starts, max_len=n)
    assert torch.equal(w[-tail:], vad.window_attention(short, short, short, 50, 4, starts=inner))
    del w
    y = vad.layer_norm(x.view(-1, dim))
    assert torch.equal(y[-5:], vad.layer_norm(x.view(-1, dim)[-5:].clone()))
    del y, x
    # a cache whose last slots lie past 2^31 elements; one key stands out, its value is the answer
    slots = 1_050_000
    ck, cv = (torch.zeros(1, slots, heads, dim, dtype=torch.bfloat16, device='cuda') for _ in range(2))
    q = torch.ones(1, heads, dim, dtype=torch.bfloat16, device='cuda')
    ck[0, slots - 3], cv[0, slots - 3] = 8.0, torch.arange(heads * dim, device='cuda').view(heads, dim).bfloat16()
    new = torch.zeros(1, heads, dim, dtype=torch.bfloat16, device='cuda')
    pos = torch.tensor([3 * slots - 2], device='cuda')
    o = vad.window_attention_step(q, new, new, ck, cv, pos, slots)
    assert torch.allclose(o[0].float(), cv[0, slots - 3].float(), rtol=2.0 ** -7)
    # the same slots far apart in memory: a slot stride past what buffer loads take
    wide = torch.zeros(70, 1, 300, 140, 128, dtype=torch.bfloat16, device='cuda')[:, 0].transpose(0, 1)[:1]
    near = wide[:, :, :heads]
    assert near.stride(1) >= 1 << 22
    ka = near.clone()
    pos = torch.tensor([40], device='cuda')
    qq, kk = _rand(g, 1, heads, dim, dtype=torch.bfloat16), _rand(g, 1, heads, dim, dtype=torch.bfloat16)
    far_o = vad.window_attention_step(qq, kk, kk, near, near.clone(), pos, 70)
    assert torch.equal(far_o, vad.window_attention_step(qq, kk, kk, ka, ka.clone(), pos, 70)) and torch.equal(near, ka)


def test_hints_windows_and_strides_at_their_ends(vad):
    """A hint shorter than the sequences, a window longer than any, one key head for all, expanded rows, rows far apart."""
    g = _gen(51)
    q, k, v, do = (_rand(g, 700, 3, 40) for _ in range(4))
    starts = torch.tensor([0, 600, 700], device='cuda')
    log_decay = _decays(3)

    def run(q, k, v, **hint):
        leaf = [t.detach().requires_grad_() for t in (q, k, v)]
        o, s = vad.linear_attention(*leaf, log_decay, starts=starts, **hint)
        outs = [o, s, *torch.autograd.grad(o, leaf, do)]
        for window, sinks in ((90, 5), (1 << 30, 0), (1 << 30, 64), (1, 0), (1, 17)):
            w = vad.window_attention(*leaf, window, sinks, starts=starts, **hint)
            outs += [w, *torch.autograd.grad(w, leaf, do)]
        return outs

    want = run(q, k, v)
    for hint in (0, 1, 65, 600, 10 ** 12):
        for a, b in zip(run(q, k, v, max_len=hint), want):
            assert torch.allclose(a, b, rtol=1e-4, atol=1e-4)
    # every window of a whole sequence and more is the same causal attention, sinks or not
    for a, b in zip(want[9:13], want[13:17]):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4)
    # a window of one row without sinks answers with that row's value.  Its weight p is 2 to the rounding error of s - max, not 1
    # to the bit, so the answer is (p v) (1 / p): half a unit for either product, a whole one for the reciprocal, 2^-24 (1 + 1 + 2)
    assert ((want[17] - v).abs() <= 2.0 ** -22 * v.abs()).all()
    # keys and values expanded over heads (stride 0): the gradient of the shared head is the heads' sum
    one = _rand(g, 700, 1, 40).requires_grad_()
    wide = one.detach().expand(700, 3, 40).clone().requires_grad_()
    a = torch.autograd.grad(vad.window_attention(q, one.expand(700, 3, 40), one.expand(700, 3, 40), 90, 5, starts=starts), one, do)[0]
    b = torch.autograd.grad(vad.window_attention(q, wide, wide, 90, 5, starts=starts), wide, do)[0]
    c = torch.autograd.grad(vad.window_attention(q, one, one, 90, 5, starts=starts), one, do)[0]
    assert torch.allclose(a, b.sum(1, keepdim=True), rtol=1e-4, atol=1e-4) and torch.allclose(a, c, rtol=1e-4, atol=1e-4)
    # one row for all rows
    row = _rand(g, 1, 3, 40).expand(700, 3, 40)
    for x, y in zip(run(row, row, row), run(*[row.contiguous()] * 3)):
        assert torch.equal(x, y)
    assert torch.equal(vad.layer_norm(row), vad.layer_norm(row.contiguous()))
    # rows farther apart than a kernel's offsets reach are brought together first
    far = torch.empty(4, 1 << 22, device='cuda').as_strided((1, 4, 3, 40), (0, 1 << 22, 40, 1))
    far.copy_(q[None, :4])
    assert torch.equal(vad.window_attention(far, far, far, 2), vad.window_attention(*[q[None, :4]] * 3, 2))
    assert torch.equal(vad.linear_attention(far, far, far, log_decay)[0], vad.linear_attention(*[q[None, :4]] * 3, log_decay)[0])
    empty = torch.empty(0, 40, device='cuda', requires_grad=True)
    w, b = torch.ones(40, device='cuda', requires_grad=True), torch.zeros(40, device='cuda', requires_grad=True)
    assert all(not t.any() for t in torch.autograd.grad(vad.layer_norm(empty, w, b).sum(), (w, b)))


@pytest.mark.parametrize('dim,window,sinks', [(40, 300, 5), (30, 256, 0), (64, 1000, 64)])
def test_large_launches_agree_with_small_ones(vad, dim, window, sinks):
    """Many rows take wider blocks than few do.  Either form is off by 2^-8 of every weight's term and of the result."""
    g = _gen(101)
    n = 8200
    q, k, v = (_rand(g, 2, n, heads, dim, dtype=torch.bfloat16) for heads in (17, 1, 1))
    k[:, 8000:], v[:, 8100:] = math.nan, math.inf
    o = vad.window_attention(q, k, v, window, sinks)
    alone = torch.cat([vad.window_attention(q[i:i + 1], k[i:i + 1], v[i:i + 1], window, sinks) for i in range(2)])
    size = vad.window_attention(q[:, :8000], k[:, :8000], v[:, :8000].abs(), window, sinks).float()
    a, b = o[:, :8000].float(), alone[:, :8000].float()
    assert ((a - b).abs() <= 2.0 ** -7 * (size * (1 + 2.0 ** -6) + b.abs())).all()
    assert o[:, 8000:].isnan().all() and alone[:, 8000:].isnan().all()
    starts = torch.tensor([0, n, 2 * n], device='cuda')
    packed = vad.window_attention(q.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), window, sinks, starts=starts, max_len=n)
    assert torch.equal(packed.view_as(o).nan_to_num(), o.nan_to_num())


def test_many_short_sequences(vad):
    """65535 sequences of 0 .. 2 rows without a hint: more tiles than a launch holds."""
    n = 65535
    lengths = torch.arange(n) % 3
    starts = torch.cat((torch.zeros(1, dtype=torch.int64), lengths.cumsum(0))).cuda()
    rows = int(starts[-1])
    g = _gen(61)
    q, k, v, do = (_rand(g, rows, 2, 4) for _ in range(4))
    leaf = [t.requires_grad_() for t in (q, k, v)]
    o = vad.window_attention(*leaf, 7, 1, starts=starts)
    grads = torch.autograd.grad(o, leaf, do)
    first = (starts[:-1][lengths.cuda() > 0])
    assert torch.allclose(o[first], v[first], rtol=1e-6, atol=1e-6)
    pairs = first[1::2]                                     # sequences of two rows
    sc = (q[pairs + 1][:, None] * torch.stack((k[pairs], k[pairs + 1]), 1)).sum(-1, keepdim=True) / 2
    want = (torch.softmax(sc, 1) * torch.stack((v[pairs], v[pairs + 1]), 1)).sum(1)
    assert torch.allclose(o[pairs + 1], want, rtol=1e-5, atol=1e-5)
    short = torch.tensor([0, 0, 1, 3], device='cuda')
    cut = [t.detach()[:3].clone().requires_grad_() for t in (q, k, v)]
    cut_grads = torch.autograd.grad(vad.window_attention(*cut, 7, 1, starts=short), cut, do[:3])
    assert all(torch.allclose(a[:3], b, rtol=1e-5, atol=1e-5) for a, b in zip(grads, cut_grads))
    o, s = vad.linear_attention(*leaf, _decays(2), starts=starts)
    assert torch.allclose(s[1], k[0][:, :, None] * v[0][:, None, :], rtol=1e-6, atol=1e-6) and not s[0].any()
    with pytest.raises(vad.VadError, match='sequence count'):
        vad.window_attention(*[torch.zeros(1, 2, 4, device='cuda')] * 3, 7, starts=torch.zeros(65537, dtype=torch.int64, device='cuda'))


def test_in_place_updates_are_seen_by_autograd(vad):
    """A state or cache that a graph has saved and a step has overwritten since: an error, not a wrong gradient."""
    g = _gen(71)
    x = _rand(g, 1, 5, 2, 8).requires_grad_()
    row = x.detach()[:, 0]
    log_decay = _decays(2)
    state = torch.zeros(1, 2, 8, 8, device='cuda')
    o, _ = vad.linear_attention(x, x, x, log_decay, state=state)
    vad.linear_attention_step(row, row, row, log_decay, state)
    with pytest.raises(RuntimeError, match='inplace'):
        o.sum().backward()
    ck, cv = (_rand(g, 1, 5, 2, 8) for _ in range(2))
    pos = torch.tensor([9], device='cuda')
    for write in (lambda: vad.window_attention_step(row, row, row, ck, cv, pos, 4, 1),
                  lambda: vad.window_cache_fill(x.detach(), x.detach(), ck, cv, 4, 1)):
        o = vad.window_attention(x, ck, cv, 4, 1)
        write()
        with pytest.raises(RuntimeError, match='inplace'):
            o.sum().backward()
    with torch.inference_mode():
        s, c, d = (torch.zeros(*n, device='cuda') for n in ((1, 2, 8, 8), (1, 5, 2, 8), (1, 5, 2, 8)))
        vad.linear_attention_step(row, row, row, log_decay, s)
        vad.window_attention_step(row, row, row, c, d, vad.window_cache_fill(x, x, c, d, 4, 1), 4, 1)
        assert s.any() and c.any()


def test_two_streams_at_once(vad):
    """The same calls on two streams at the same time, each with its own tensors and scratch memory."""
    def work(seed):
        g = _gen(seed)
        q, k, v, do = (_rand(g, 4000, 4, 64, dtype=torch.bfloat16) for _ in range(4))
        leaf = [t.requires_grad_() for t in (q, k, v)]
        log_decay = _decays(4)
        cache = torch.zeros(2, 1, 4016, 4, 64, dtype=torch.bfloat16, device='cuda')

        def run():
            o, s = vad.linear_attention(*leaf, log_decay, starts=starts)
            w = vad.window_attention(*leaf, 200, 16, starts=starts)
            grads = (*torch.autograd.grad(o, leaf, do), *torch.autograd.grad(w, leaf, do))
            with torch.no_grad():
                pos = vad.window_cache_fill(k[None], v[None], cache[0], cache[1], 4000, 16)
                step = vad.window_attention_step(q[:1], k[:1], v[:1], cache[0], cache[1], pos, 4000, 16)
            return [o, s, w, *grads, step]
        return run

    starts = torch.tensor([0, 3000, 4000], device='cuda')
    runs = [work(81), work(82)]
    want = [[t.clone() for t in run()] for run in runs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for run, stream in zip(runs, streams):
            with torch.cuda.stream(stream):
                got.append(run())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_nothing_is_written_behind_a_head(vad):
    """Caches, states and outputs of head sizes that end inside a 16-byte piece, between guard values."""
    g = _gen(41)
    for dtype in DTYPES:
        for dim in (1, 2, 3, 6, 7, 30, 33, 66):
            q, k, v = (_rand(g, 2, 2, dim, dtype=dtype) for _ in range(3))
            room = torch.full((2, 2, 9, 2, dim + 8), 7.0, dtype=dtype, device='cuda')
            ck, cv = room[0, ..., :dim], room[1, ..., :dim]
            pos = vad.window_cache_fill(*(_rand(g, 2, 12, 2, dim, dtype=dtype) for _ in range(2)), ck, cv, 8, 1)
            for _ in range(3):
                vad.window_attention_step(q, k, v, ck, cv, pos, 8, 1)
                pos += 1
            assert (room[..., dim:] == 7.0).all()


def test_a_streaming_model_scores_frames_as_it_scores_the_recording(vad):
    """The operators together: norm -> linear attention -> norm -> window attention over features of synthetic audio, trained
    for a gradient over the whole recording, then run frame by frame from where the recording stopped."""
    torch.manual_seed(0)
    frames, heads, dim, window, sinks = 160, 3, 30, 30, 2
    feat = vad.mfcc_delta_stream(vad.synth_stream(0, frames, seed=5), frames)
    width = heads * dim
    shapes = [(24, 3 * width), (width, 3 * width), (width, 2)]
    params = [(torch.randn(s, device='cuda') / s[0] ** 0.5).requires_grad_() for s in shapes]
    gains = [torch.ones(n, device='cuda', requires_grad=True) for n in (24, width)]
    shifts = [torch.zeros(n, device='cuda', requires_grad=True) for n in (24, width)]
    log_decay = _decays(heads)

    def split(x, p):
        return (x @ p).unflatten(-1, (3, heads, dim)).unbind(-3)

    def model(x, layer_norm, mix, look):
        h = mix(*split(layer_norm(x, gains[0], shifts[0]), params[0])).flatten(-2)
        h = h + look(*split(layer_norm(h, gains[1], shifts[1]), params[1])).flatten(-2)
        return h @ params[2]

    def plain_mix(q, k, v):
        return torch.stack([ref.decay_sequence(q[0, :, i], k[0, :, i], v[0, :, i], float(a), dim ** -0.5)['o']
                            for i, a in enumerate(log_decay.clamp(-87.0, 0.0).double())], 1)[None]

    def plain_look(q, k, v):
        return torch.stack([ref.window_sequence(q[0, :, i], k[0, :, i], v[0, :, i], window, sinks, dim ** -0.5)['o'] for i in range(heads)], 1)[None]

    leaves = params + gains + shifts
    scores = model(feat[None], vad.layer_norm, lambda *t: vad.linear_attention(*t, log_decay)[0], lambda *t: vad.window_attention(*t, window, sinks))
    grads = torch.autograd.grad(torch.logsumexp(scores, -1).sum() - scores[..., 1].sum(), leaves)
    saved = [p.data for p in leaves]
    for p in leaves:
        p.data = p.data.double()
    want = model(feat[None].double(), lambda x, w, b: ref.layer_norm(x, w, b, 1e-5), plain_mix, plain_look)
    wants = torch.autograd.grad(torch.logsumexp(want, -1).sum() - want[..., 1].sum(), leaves)
    for p, d in zip(leaves, saved):
        p.data = d
    # float32 through two mixers and two norms: thousands of roundings of 2^-24 against the largest value
    assert float((scores.double() - want).detach().abs().max()) < 1e-3 * float(want.detach().abs().max())
    for a, b in zip(grads, wants):
        assert float((a.double() - b).abs().max()) < 1e-3 * float(b.abs().max())

    live, state, cache = 130, {}, {}
    with torch.no_grad():
        def start_mix(q, k, v):
            o, state['s'] = vad.linear_attention(q, k, v, log_decay)
            return o

        def start_look(q, k, v):
            cache['k'], cache['v'] = (torch.empty(1, sinks + window, heads, dim, device='cuda') for _ in range(2))
            cache['pos'] = vad.window_cache_fill(k, v, cache['k'], cache['v'], window, sinks)
            return vad.window_attention(q, k, v, window, sinks)

        head = model(feat[None, :live], vad.layer_norm, start_mix, start_look)
        assert torch.allclose(head[0], scores[0, :live], rtol=1e-4, atol=1e-4)
        for t in range(live, frames):
            step = model(feat[t:t + 1], vad.layer_norm, lambda *x: vad.linear_attention_step(*x, log_decay, state['s']),
                         lambda *x: vad.window_attention_step(*x, cache['k'], cache['v'], cache['pos'], window, sinks))
            cache['pos'] += 1
            assert torch.allclose(step[0], scores[0, t], rtol=1e-3, atol=1e-3)


def test_device_refusals(vad):
    """Refusals that need device tensors to reach: nothing is launched."""
    q = torch.zeros(1, 10, 4, 32, device='cuda')
    ld = torch.zeros(4, device='cuda')
    bad = [
        (lambda: vad.layer_norm(q.double()), 'float32 or bfloat16'),
        (lambda: vad.layer_norm(q, torch.ones(31, device='cuda')), 'shape'),
        (lambda: vad.layer_norm(q, torch.ones(32, device='cuda'), torch.ones(32, device='cuda').bfloat16()), 'float32'),
        (lambda: vad.layer_norm(q, eps=float('nan')), 'eps'),
        (lambda: vad.layer_norm(torch.zeros((), device='cuda')), 'last dimension'),
        (lambda: vad.linear_attention(q, q, q[:, :9], ld), 'go together'),
        (lambda: vad.linear_attention(q, q.bfloat16(), q, ld), 'k must be'),
        (lambda: vad.linear_attention(q, q[:, :, :2], q[:, :, :2], ld), 'query heads'),
        (lambda: vad.linear_attention(q, q, q, ld[:3]), 'log_decay'),
        (lambda: vad.linear_attention(q, q, q, ld.requires_grad_()), 'no gradient'),
        (lambda: vad.linear_attention(q, q, q, torch.zeros(4, device='cuda'), state=torch.zeros(1, 4, 32, 31, device='cuda')), 'state'),
        (lambda: vad.linear_attention(q, q, q, torch.zeros(4, device='cuda'), scale=float('inf')), 'scale'),
        (lambda: vad.linear_attention(q, q, q, torch.zeros(4, device='cuda'), starts=torch.zeros(2, dtype=torch.int64, device='cuda')), 'rows, heads'),
        (lambda: vad.linear_attention(q[0], q[0], q[0], torch.zeros(4, device='cuda'), starts=torch.zeros(2, device='cuda')), 'starts'),
        (lambda: vad.linear_attention(q[0], q[0], q[0], torch.zeros(4, device='cuda'), starts=torch.zeros(0, dtype=torch.int64, device='cuda')), 'starts'),
        (lambda: vad.linear_attention_step(q[0], q[0], q[0], torch.zeros(4, device='cuda'), torch.zeros(10, 4, 32, 32, device='cuda').mT), 'contiguous'),
        (lambda: vad.window_attention(q, q, q, 0), 'window'),
        (lambda: vad.window_attention(q, q, q, 5, 65), 'sinks'),
        (lambda: vad.window_attention(q, q, q, 5, scale=-1.0), 'scale'),
        (lambda: vad.window_attention(q, q[:, :, :3], q[:, :, :3], 5), 'query heads'),
        (lambda: vad.window_attention(torch.zeros(1, 2, 1, 129, device='cuda'), *[torch.zeros(1, 2, 1, 129, device='cuda')] * 2, 5), 'dim'),
        (lambda: vad.window_attention_step(q[0], q[0], q[0], *[torch.zeros(10, 6, 4, 32, device='cuda')] * 2, torch.zeros(10, device='cuda'), 5, 1), 'pos'),
        (lambda: vad.window_attention_step(q[0], q[0], q[0], *[torch.zeros(10, 5, 4, 32, device='cuda')] * 2, torch.zeros(10, dtype=torch.int64, device='cuda'), 5, 1), 'cache_k'),
        (lambda: vad.window_attention_step(q[0], q[0], q[0], torch.zeros(10, 6, 4, 32, device='cuda'), torch.zeros(1, 6, 4, 32, device='cuda').expand(10, 6, 4, 32),
                                           torch.zeros(10, dtype=torch.int64, device='cuda'), 5, 1), 'broadcast'),
        (lambda: vad.window_cache_fill(q, q, *[torch.zeros(1, 6, 4, 32, device='cuda')] * 2, 5, 1), 'same memory'),
        (lambda: vad.window_cache_fill(q.clone().requires_grad_(), q, *[torch.zeros(1, 6, 4, 32, device='cuda') for _ in range(2)], 5, 1), 'no gradient'),
    ]
    for call, needle in bad:
        with pytest.raises(ValueError, match=needle):
            call()
    with pytest.raises(ValueError, match='no gradient'):
        vad.linear_attention_step(q[0].clone().requires_grad_(), q[0], q[0], torch.zeros(4, device='cuda'), torch.zeros(10, 4, 32, 32, device='cuda'))
    leaf = q.clone().requires_grad_()
    first = torch.autograd.grad(vad.layer_norm(leaf).square().sum(), leaf, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), leaf)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('window,sinks', [(129, 0), (190, 3), (650, 64)])
def test_window_step_with_infinities_in_the_new_row(vad, dtype, window, sinks):
    """An infinite value in the new row reaches the output as that infinity from every slot, those next to the ends of the
    parts that a cache is cut into among them; the other columns stay finite."""
    g = _gen(window)
    slots, dim = sinks + window, 128
    ck, cv = (_rand(g, 1, slots, 2, dim, dtype=dtype) for _ in range(2))
    q = _rand(g, slots, 2, dim, dtype=dtype)
    k, v = (_rand(g, slots, 2, dim, dtype=dtype) for _ in range(2))
    v[:, :, 3], v[:, :, 70] = math.inf, -math.inf
    rest = torch.ones(dim, dtype=torch.bool, device='cuda')
    rest[3] = rest[70] = False
    for slot in range(sinks, slots):
        pos = torch.tensor([slot + window], device='cuda')
        kk, vv = ck.clone(), cv.clone()
        i = slice(slot, slot + 1)
        o = vad.window_attention_step(q[i], k[i], v[i], kk, vv, pos, window, sinks)[0].float()
        assert (o[:, 3] == math.inf).all() and (o[:, 70] == -math.inf).all(), slot
        p = torch.softmax((kk[0].double() * q[i].double()).sum(-1) * dim ** -0.5, 0)              # slots, heads
        want = (p[..., None] * vv[0].double())[..., rest].sum(0)
        assert float((o[:, rest].double() - want).abs().max()) < 1e-5 + 2 * U[dtype] * float(want.abs().max()), slot


def _outer_sums(keys, values, queries, a, scale, back=False):
    """S_t = a S_{t-1} + keys_t values_t^T row by row, o_t = scale queries_t S_t, one product at a time in float64; `back`: from
    the last row to the first.  The S behind the last row taken and the rows o."""
    s, out = torch.zeros(keys.size(1), values.size(1), dtype=torch.float64, device=keys.device), []
    order = range(keys.size(0))
    for t in reversed(order) if back else order:
        s = a * s + keys[t, :, None] * values[t, None, :]
        out.append(scale * (queries[t, :, None] * s).sum(0))
    return s, torch.stack(out[::-1] if back else out)


def _same_kinds(got, want, what):
    """Infinities of the same sign, NaN and finite values in the same places."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), what
    for sign in (math.inf, -math.inf):
        assert torch.equal(got == sign, want == sign), what


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('length,dim', [(50, 64), (150, 30), (1000, 64), (300, 128)])
def test_linear_attention_infinite_keys(vad, dtype, length, dim):
    """An infinite key makes infinities of the state's row and of what its queries read, NaN only where the recurrence itself has
    one; infinite output gradients do the same to dk, in either type."""
    g = _gen(length + dim)
    # values that a few bits hold and no product that vanishes: the lower terms of a split float32 are zero
    q, k, v, do = (torch.randint(1, 5, (1, length, 2, dim), generator=g, device='cuda').to(dtype) / 4 for _ in range(4))
    signs = torch.randint(0, 2, (4, 1, length, 2, dim), generator=g, device='cuda') * 2 - 1
    q, k, v, do = (t * s for t, s in zip((q, k, v, do), signs))
    log_decay = torch.tensor([0.0, -0.01], device='cuda')

    def spoilt(t):
        bad = t.clone()
        bad[0, 20, 0, 5], bad[0, length - 3, 1, dim - 1] = math.inf, -math.inf
        return bad

    bad = spoilt(k)
    o, s = vad.linear_attention(q, bad, v, log_decay, scale=0.5)
    leaf = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(vad.linear_attention(*leaf, log_decay, scale=0.5)[0], leaf, spoilt(do))
    for h, a in enumerate(log_decay.double().exp().tolist()):
        x = [t[0, :, h].double() for t in (q, bad, v, spoilt(do))]
        ws, wo = _outer_sums(x[1], x[2], x[0], a, 0.5)
        assert ws.isinf().any() and not ws.isnan().any()
        _same_kinds(s[0, h], ws, 'state')
        _same_kinds(o[0, :, h], wo, 'o')
        _same_kinds(grads[1][0, :, h], _outer_sums(x[3], x[0], x[2], a, 0.5, back=True)[1], 'dk')


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('length,dim', [(50, 64), (150, 30), (1000, 70), (300, 128)])
def test_linear_attention_infinite_values(vad, dtype, length, dim):
    """An infinite value where nothing is negative is an infinity in the state's column and in the rows behind it, and one of the
    output's gradient is one in dv, at any head size: no order of the sums makes NaN of it."""
    g = _gen(length + dim)
    q, k, v, do = (torch.randint(1, 5, (1, length, 2, dim), generator=g, device='cuda').to(dtype) / 4 for _ in range(4))
    log_decay = torch.tensor([0.0, -0.01], device='cuda')
    bad, bad_do = v.clone(), do.clone()
    bad[0, 20, 0, 5], bad[0, length - 3, 1, dim - 1] = math.inf, math.inf
    bad_do[0, length - 20, 0, 5], bad_do[0, 2, 1, dim - 1] = math.inf, math.inf
    o, s = vad.linear_attention(q, k, bad, log_decay, scale=0.5)
    leaf = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(vad.linear_attention(*leaf, log_decay, scale=0.5)[0], leaf, bad_do)
    for h, a in enumerate(log_decay.double().exp().tolist()):
        x = [t[0, :, h].double() for t in (q, k, bad, bad_do)]
        ws, wo = _outer_sums(x[1], x[2], x[0], a, 0.5)
        assert ws.isinf().any() and not ws.isnan().any() and not wo.isnan().any()
        _same_kinds(s[0, h], ws, 'state')
        _same_kinds(o[0, :, h], wo, 'o')
        _same_kinds(grads[2][0, :, h], _outer_sums(x[0], x[3], x[1], a, 0.5, back=True)[1], 'dv')


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [30, 64, 128])
def test_infinities_are_found_in_every_column(vad, dtype, dim):
    """One infinity or NaN per sequence, each in another column, of k and of v."""
    g = _gen(dim)
    n = torch.arange(dim, device='cuda')
    q, k, v = (torch.randint(1, 5, (dim, 70, 1, dim), generator=g, device='cuda').to(dtype) / 4 for _ in range(3))
    log_decay = torch.tensor([-0.01], device='cuda')
    for value in (math.inf, -math.inf, math.nan):
        kk, vv = k.clone(), v.clone()
        kk[n, n * 7 % 64, 0, n] = value
        vv[n, n * 5 % 64, 0, n] = value
        for a, b, axis, row in ((kk, v, 1, n * 7 % 64), (k, vv, 2, n * 5 % 64)):
            o, s = vad.linear_attention(q, a, b, log_decay)
            hit = torch.zeros(dim, dim, dim, dtype=torch.bool, device='cuda')
            hit[n, n] = True
            hit = hit if axis == 1 else hit.transpose(1, 2)
            want = torch.full_like(s[:, 0], value)
            assert torch.equal(s[:, 0].isfinite(), ~hit)
            assert torch.equal(s[:, 0][hit].isnan(), want[hit].isnan()) and (value != value or torch.equal(s[:, 0][hit], want[hit]))
            w = vad.window_attention(q, a, b, 20)
            assert torch.isfinite(w[row < 50, 69]).all() and not torch.isfinite(o[:, 69]).all()


def test_derivatives_and_recordings_that_cannot_pass_are_refused(vad):
    """Forward-mode derivatives, also of an output's gradient, and calls that a tracer would not record: an error in place of a
    result that lacks them.  Plain tensors in a dual level are computed."""
    g = _gen(5)
    q, k, v = (_rand(g, 1, 10, 2, 16) for _ in range(3))
    log_decay = _decays(2)
    calls = [lambda x: vad.layer_norm(x), lambda x: vad.linear_attention(x, k, v, log_decay)[0], lambda x: vad.window_attention(x, k, v, 4)]
    with forward_ad.dual_level():
        for call in calls:
            for x in (q, q.clone().requires_grad_()):
                with pytest.raises(ValueError, match='forward-mode'):
                    call(forward_ad.make_dual(x, torch.ones_like(x)))
            leaf = q.clone().requires_grad_()
            o = call(leaf)
            assert forward_ad.unpack_dual(o).tangent is None
            with pytest.raises(ValueError, match='forward-mode'):
                torch.autograd.grad(o, leaf, forward_ad.make_dual(torch.ones_like(o), torch.ones_like(o)))
    row, pos = q[0], torch.zeros(10, dtype=torch.int64, device='cuda')
    state, cache = torch.zeros(10, 2, 16, 16, device='cuda'), torch.zeros(2, 10, 4, 2, 16, device='cuda')
    one = torch.zeros(2, 1, 4, 2, 16, device='cuda')
    calls += [lambda x: vad.linear_attention_step(x[0], row, row, log_decay, state),
              lambda x: vad.window_attention_step(x[0], row, row, cache[0], cache[1], pos, 4), lambda x: vad.window_cache_fill(x, v, one[0], one[1], 4)]
    for call in calls:
        with pytest.raises(ValueError, match='traced'):
            torch.jit.trace(call, (q,), check_trace=False)
        with pytest.raises(ValueError, match='traced'):
            make_fx(call)(q)
    assert not state.any() and not cache.any() and not one.any()
    for transform in (lambda call: torch.vmap(call)(q[None]), lambda call: torch.func.jvp(call, (q,), (q,)),
                      lambda call: torch.func.grad(lambda x: call(x).sum())(q)):
        for call in calls[:3]:
            with pytest.raises((RuntimeError, ValueError)):
                transform(call)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('cols', [30, 900, 1024, 1025, 5000, 20001])
def test_layer_norm_of_far_rows(vad, dtype, cols):
    """Rows far from zero: the mean's own rounding stays out of the deviations, in either direction.  A sum of n terms of size s is
    off by at most n 2^-24 s; taken again over the deviations, what is left of the mean's error is n 2^-24 of them and, of the
    offset, (n 2^-24)^2."""
    g = _gen(cols)
    n = (cols / 64 + 10 if cols <= 4096 else 180) * ULP               # values down a lane and levels across, as in test_layer_norm
    w, b = 1 + _rand(g, cols, scale=0.3), _rand(g, cols)
    for offset in (1e2, 1e4, 1e6):
        x = (_rand(g, 6, cols) + offset).to(dtype)
        x[0], x[1], x[2] = offset, offset + 0.3, -1.37 * offset       # no variance
        x, w, b = (t.detach().requires_grad_() for t in (x, w, b))
        dy = _rand(g, 6, cols, dtype=dtype)
        y = vad.layer_norm(x, w, b)
        grads = torch.autograd.grad(y, (x, w, b), dy)
        want = ref.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5, dy)
        xd = x.detach().double()
        c = xd - xd.mean(1, keepdim=True)
        r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5)
        xh = (c * r).abs()
        # deviations off by n of their mean size and by their own rounding; r by the same, relatively, three roundings more
        mag_xh = xh.mean(1, keepdim=True) + 8 * xh + n * xd.abs().amax(1, keepdim=True) * r
        _close(y.detach(), want[0], mag_xh * w.detach().abs() + b.detach().abs(), 2 * n, dtype, 'y at %g' % offset)
        gw = (dy.double() * w.detach()).abs()
        mag = r * (gw + gw.mean(1, keepdim=True) + (xh + mag_xh) * (gw * (xh + mag_xh)).mean(1, keepdim=True)) * 4
        _close(grads[0], want[1], mag, 2 * n, dtype, 'dx at %g' % offset)
        _close(grads[1], want[2], (dy.double().abs() * (xh + mag_xh)).sum(0), 2 * n + 70 * ULP, torch.float32, 'dw at %g' % offset)


@pytest.mark.parametrize('dtype', DTYPES)
def test_single_rows_of_any_stride(vad, dtype):
    """One row has no row stride, whatever its tensor says: a slice of a longer batch, one frame of many channels kept time first,
    heads laid out behind the row."""
    g = _gen(15)
    log_decay = torch.tensor([-0.1], device='cuda').expand(64).contiguous()
    wide = torch.zeros(2, 8192, 16, 64, dtype=dtype, device='cuda')[0:1, 0]
    frame = torch.zeros(1, 8192, 32, 16, dtype=dtype, device='cuda').transpose(0, 1)
    inside = torch.zeros(3, 4, 32, 1, dtype=dtype, device='cuda').permute(0, 3, 1, 2)
    assert wide.stride(0) >= 1 << 22 and frame.stride(1) >= 1 << 22 and inside.stride(1) == 1
    for t in (wide, frame, inside):
        t.copy_(_rand(g, *t.shape, dtype=dtype))
        starts = torch.tensor([0, 1], device='cuda') if t.dim() == 3 else None
        heads, dim, n = t.size(-2), t.size(-1), 1 if t.dim() == 3 else t.size(0)

        def run(x, gy):
            leaf = [x.detach().requires_grad_() for _ in range(3)]
            o, s = vad.linear_attention(*leaf, log_decay[:heads], starts=starts)
            w = vad.window_attention(*leaf, 5, 1, starts=starts)
            ck, cv = (torch.zeros(n, 6, heads, dim, dtype=dtype, device='cuda') for _ in range(2))
            with torch.no_grad():
                pos = vad.window_cache_fill(x, x, ck, cv, 5, 1, starts=starts)
            return [o, s, w, ck, cv, pos, *torch.autograd.grad(o, leaf, gy), *torch.autograd.grad(w, leaf, gy)]

        plain = t.clone(memory_format=torch.contiguous_format)
        plain = plain.as_strided(plain.shape, torch.empty(plain.shape).stride())
        for a, b in zip(run(t, t), run(plain, plain)):
            assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', DTYPES)
def test_caches_of_one_slot_at_any_stride(vad, dtype):
    """A cache of one slot has no slot stride: what the slot held before, NaN here, does not come back as that of a next one."""
    g = _gen(16)
    q, k, v = (_rand(g, 3, 2, 64, dtype=dtype) for _ in range(3))
    pos = torch.tensor([0, 5, 9], device='cuda')
    caches = [torch.full((3, 2, 64, 1), math.nan, dtype=dtype, device='cuda').permute(0, 3, 1, 2) for _ in range(2)]
    caches += [torch.full((3, 2, 64), math.nan, dtype=dtype, device='cuda').as_strided((3, 1, 2, 64), (128, 0, 64, 1)) for _ in range(2)]
    assert caches[0].stride(1) == 1
    for ck, cv in (caches[:2], caches[2:]):
        o = vad.window_attention_step(q, k, v, ck, cv, pos, 1)
        assert torch.equal(o, v) and torch.equal(ck[:, 0], k) and torch.equal(cv[:, 0], v)


@pytest.mark.parametrize('dtype', DTYPES)
def test_overlapping_rows(vad, dtype):
    """One row for all, and rows that share memory, reach no further than copies of them: an infinite key stays one infinity in the
    state's row."""
    g = _gen(17)
    n, dim = 70, 64
    log_decay = torch.zeros(1, device='cuda')
    q, v = (_rand(g, 1, n, 1, dim, dtype=dtype).abs() + 0.5 for _ in range(2))
    row = _rand(g, 1, 1, 1, dim, dtype=dtype)
    row[..., 7] = math.inf
    run = _rand(g, n + dim, dtype=dtype)
    run[3 * dim // 2] = math.inf
    for k in (row.expand(1, n, 1, dim), run.as_strided((1, n, 1, dim), (n + dim, 1, dim, 1))):
        for got, want in zip(vad.linear_attention(q, k, v, log_decay), vad.linear_attention(q, k.contiguous(), v, log_decay)):
            assert torch.equal(got.nan_to_num(), want.nan_to_num()) and torch.equal(got.isnan(), want.isnan())
        s = vad.linear_attention(q, k, v, log_decay)[1]
        assert s.isinf().any() and not s.isnan().any()
        # the entry point itself, which Python calls with copies of such rows
        L, strides = vad.lib(), [(ctypes.c_int64 * 3)(*t.stride()[:3]) for t in (q, k, v)]
        size = L.vad_linear_attention_workspace_bytes(1, n, 1, dim, 0)
        ws, o, state = torch.empty(size, dtype=torch.uint8, device='cuda'), torch.empty_like(v), torch.empty_like(s)
        rc = L.vad_linear_attention_forward(q.data_ptr(), strides[0], k.data_ptr(), strides[1], v.data_ptr(), strides[2], None, 1, 0, n, 1, dim,
                                            dtype is torch.bfloat16, log_decay.data_ptr(), dim ** -0.5, None, o.data_ptr(), state.data_ptr(),
                                            ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and torch.equal(state, s) and torch.equal(o.nan_to_num(), vad.linear_attention(q, k, v, log_decay)[0].nan_to_num())
        for got, want in zip(vad.linear_attention(q, v, k, log_decay), vad.linear_attention(q, v, k.contiguous(), log_decay)):
            assert torch.equal(got.nan_to_num(), want.nan_to_num()) and torch.equal(got.isnan(), want.isnan())


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('at', [3, 100, 200])
def test_window_attention_infinite_keys_in_dq(vad, dtype, at):
    """A key with an infinity has a score of an infinity or NaN for every row that sees it.  Where that is minus infinity its weight
    is zero and dS K is zero times infinity, wherever the key stands in its tile; rows that do not see it stay finite."""
    g = _gen(18)
    n, window, sinks = 300, 90, 4
    q, do = (_rand(g, 1, n, 2, 64, dtype=dtype).abs() + 0.1 for _ in range(2))
    k, v = (_rand(g, 1, n, 1, 64, dtype=dtype) for _ in range(2))
    k[0, at, 0, 9] = -math.inf
    leaf = [t.requires_grad_() for t in (q, k, v)]
    o = vad.window_attention(*leaf, window, sinks)
    dq = torch.autograd.grad(o, leaf, do)[0]
    rows = torch.arange(n, device='cuda')
    sees = (rows >= at) & ((rows - at < window) | (at < sinks)) & (rows > 0)
    assert dq[0, sees][..., 9].isnan().all()
    others = torch.arange(64, device='cuda') != 9
    assert torch.isfinite(o).all() and torch.isfinite(dq[0, ~sees]).all() and torch.isfinite(dq[0, sees][..., others]).all()
