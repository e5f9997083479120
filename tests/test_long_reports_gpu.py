"""Rotary positions and windowed attention on the device, against their 64-bit forms within counted roundings (tests/long_report_oracle.py)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from ct_clip_amd import functional as Fn  # noqa: E402
from tests import long_report_oracle as O  # noqa: E402

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def rnd(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV).to(dtype)


# ------------------------------------------------------------------------------------------------------------------ rotary

ROTARY = [  # M, L, start, Hq, Hk, D, rot, interleaved, positions, scaling
    (1, 1, 0, 12, 12, 64, 64, False, None, None),
    (1, 1, 2 ** 40 + 7, 1, 1, 64, 64, False, None, None),
    (77, 11, 1000003, 3, 1, 32, 32, False, None, dict(type="linear", factor=4.0)),
    (1030, 515, 0, 12, 4, 64, 32, True, None, dict(type="yarn", factor=8.0, original_length=512)),
    (4100, 4100, 5, 5, 0, 128, 64, False, None, dict(type="ntk", factor=2.0)),
    (333, 333, 0, 2, 2, 64, 64, False, torch.int32, None),
    (333, 333, 0, 2, 2, 64, 48, True, torch.int64, None),
    (9, 3, 0, 3, 2, 6, 2, False, None, None),               # element-wise kernel: odd heads, rot 2
    (65, 65, 3, 2, 1, 40, 20, True, None, None),
    (50, 50, 0, 1, 1, 48, 24, False, None, None),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,L,start,Hq,Hk,D,rot,inter,posdt,scaling", ROTARY)
def test_rotary_forward_and_backward(M, L, start, Hq, Hk, D, rot, inter, posdt, scaling, dtype):
    rope = Fn.RotaryPositions(rot, layout="interleaved" if inter else "half", scaling=scaling)
    q = rnd((M, Hq * D), dtype, 1).requires_grad_(True)
    k = rnd((M, Hk * D), dtype, 2).requires_grad_(True) if Hk else None
    positions = None
    pos = start + torch.arange(M, device=DEV) % L
    if posdt is not None:
        pos = torch.randint(-5, 2 ** 31 - 1 if posdt == torch.int32 else 2 ** 45, (M,), generator=torch.Generator().manual_seed(3)).to(DEV)
        positions = pos.to(posdt)
    out = Fn.rotary(q, k, rope, D, L=L, positions=positions, start=start)
    out = out if Hk else (out,)
    xs = (q, k) if Hk else (q,)
    gs = [rnd(tuple(x.shape), dtype, 5 + i) for i, x in enumerate(xs)]
    grads = torch.autograd.grad(out, xs, gs)
    # angles of far positions in integers (64-bit floats would lose what is tested): turns modulo one, then the plain form at the remaining angle
    small = pos.abs().max().item() < 2 ** 21
    for i, x in enumerate(xs):
        if small:
            w = O.rotary64(x.detach(), torch.from_numpy(rope.frequencies), rope.magnitude, D, rot, inter, pos)
            b = O.rotary64(gs[i], torch.from_numpy(rope.frequencies), rope.magnitude, D, rot, inter, pos, inverse=True)
        else:
            w = far_rotary64(x.detach(), rope, D, rot, inter, pos, 1)
            b = far_rotary64(gs[i], rope, D, rot, inter, pos, -1)
        O.check(out[i].detach(), (w[0], O.rotary_bound(*w, dtype)), f"out {i}")
        O.check(grads[i], (b[0], O.rotary_bound(*b, dtype)), f"grad {i}")


def far_rotary64(x, rope, D, rot, inter, pos, sign):
    """Row by row: position times the 64-bit fraction of a turn in whole numbers, modulo one turn."""
    turns = torch.tensor([[((int(p) * int(b)) % 2 ** 64) / 2.0 ** 64 for b in rope.bits] for p in pos.tolist()], dtype=torch.float64, device=x.device)
    ang = turns * 2 * math.pi * sign
    y = x.double().reshape(x.shape[0], -1, D)
    c, s = torch.cos(ang)[:, None] * rope.magnitude, torch.sin(ang)[:, None] * rope.magnitude
    ia = slice(0, rot, 2) if inter else slice(0, rot // 2)
    ib = slice(1, rot, 2) if inter else slice(rot // 2, rot)
    a, b = y[..., ia], y[..., ib]
    z, m = y.clone(), torch.zeros_like(y)
    z[..., ia], z[..., ib] = a * c - b * s, b * c + a * s
    m[..., ia] = m[..., ib] = (a.abs() + b.abs()) * rope.magnitude
    return z.reshape(x.shape[0], -1), m.reshape(x.shape[0], -1)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rotary_in_place_on_the_projection_and_odd_strides(dtype):
    """Column views of one buffer, in place: the v columns stay as they were; a pitch and an offset that only the element-wise kernel serves give the same."""
    from ct_clip_amd import backend
    be, H, D, M = backend.get(), 4, 64, 150
    rope = Fn.RotaryPositions(32)
    buf = rnd((M, 3 * H * D), dtype, 9)
    want = buf.clone()
    q, k = want[:, :H * D], want[:, H * D:2 * H * D]
    nq, nk = Fn.rotary(q, k, rope, D, L=50, start=2)
    be.rotary(buf[:, :H * D], buf[:, H * D:2 * H * D], rope.turns(buf.device), D, 32, 50, None, 2, False, 1.0, out=(buf[:, :H * D], buf[:, H * D:2 * H * D]))
    assert torch.equal(buf[:, :H * D], nq) and torch.equal(buf[:, H * D:2 * H * D], nk) and torch.equal(buf[:, 2 * H * D:], want[:, 2 * H * D:])
    odd = torch.zeros((M, H * D + 3), dtype=dtype, device=DEV)
    odd[:, 1:1 + H * D] = q
    assert torch.equal(Fn.rotary(odd[:, 1:1 + H * D], None, rope, D, L=50, start=2), nq)


def test_rotary_gradient_against_differences():
    rope = Fn.RotaryPositions(32, scaling=dict(type="yarn", factor=4.0, original_length=256))
    x = rnd((7, 2 * 32), F32, 11).requires_grad_(True)
    g, d = rnd((7, 64), F32, 12), rnd((7, 64), F32, 13)
    (dx,) = torch.autograd.grad(Fn.rotary(x, None, rope, 32, start=100), x, g)
    # linear: the difference quotient is exact up to the roundings of two outputs (4 u of |y| each, y within sqrt(2) magnitude |x|, step 1/4)
    h = 0.25
    with torch.no_grad():
        num = ((Fn.rotary(x + h * d, None, rope, 32, start=100).double() - Fn.rotary(x - h * d, None, rope, 32, start=100).double()) / (2 * h) * g.double()).sum()
    room = 16 * O.U32 * 2 * ((x.detach().abs() + d.abs()).double().sum(1).max() * g.abs().double().sum()) / (2 * h)
    assert abs(num - (dx.double() * d.double()).sum()) <= room


# --------------------------------------------------------------------------------------------------------------- attention

def make_mask(kind, nseq, Lk, seed):
    if kind is None:
        return None
    j, b = torch.arange(Lk)[None, :], torch.arange(nseq)[:, None]
    m = torch.zeros((nseq, Lk))
    if kind == "pad":
        m[(j >= Lk - (b * Lk) // (2 * nseq)).expand(nseq, Lk)] = torch.finfo(F32).min
    elif kind == "holes":            # finfo.min, -inf and NaN all hide; the last sequence sees nothing
        m = torch.randn((nseq, Lk), generator=torch.Generator().manual_seed(seed))
        m[((j * 7 + b * 3) % 5 == 0).expand(nseq, Lk)] = -math.inf
        m[((j * 7 + b * 3) % 5 == 1).expand(nseq, Lk)] = math.nan
        if nseq > 1:
            m[-1] = torch.finfo(F32).min
    elif kind == "front":            # the first two thirds hidden: rows of a left-bounded window see nothing
        m[(j < 2 * Lk // 3).expand(nseq, Lk)] = torch.finfo(F32).min
    return m.to(DEV)


def run_case(dtype, nseq, Lq, Lk, H, Hk, D, window, sinks, q_start=0, mask=None, lengths=None, first=0, tail=0, drop=None, seed=0, poison=True, strided=True, grad=True):
    if lengths is not None:
        M = first + sum(lengths) + tail
        Mq = Mk = M
        spans, at = [], first
        for n in lengths:
            spans.append((at, n, at, n))
            at += n
        nseq = Fn.PackedSequences(lengths, first=first)
        keymask = make_mask(mask, 1, M, seed + 7)
    else:
        Mq, Mk = nseq * Lq, nseq * Lk
        spans = [(b * Lq, Lq, b * Lk, Lk) for b in range(nseq)]
        keymask = make_mask(mask, nseq, Lk, seed + 7)
    if strided and Mq == Mk:
        buf = rnd((Mq, (H + 2 * Hk) * D), dtype, seed + 1)
        q, k, v = buf[:, :H * D], buf[:, H * D:(H + Hk) * D], buf[:, (H + Hk) * D:]
    else:
        q, k, v = rnd((Mq, H * D), dtype, seed + 1), rnd((Mk, Hk * D), dtype, seed + 2), rnd((Mk, Hk * D), dtype, seed + 3)
    if keymask is not None and poison:       # whatever stands in a hidden key
        bad = ~(keymask.reshape(-1) > -1e30)
        k[bad] = math.nan
        v[bad] = math.inf
    q, k, v = (t.detach().requires_grad_(grad) for t in (q, k, v))
    scale = 0.9 / math.sqrt(D)
    do = rnd((Mq, H * D), dtype, seed + 4) if grad else None
    o = Fn.window_attention(q, k, v, H, D, nseq=nseq, kv_heads=Hk, window=window, sinks=sinks, keymask=keymask, scale=scale, q_start=q_start, dropout=drop)
    left, right = window if isinstance(window, tuple) else (window, window)
    mult = None
    if drop is not None:
        from ct_clip_amd import backend
        top = max(s[3] for s in spans)
        m = backend.get().attn_dropout_mask(len(spans), H, top, drop[0], drop[1], torch.device(DEV))
        mult = [m[b] for b in range(len(spans))]
    want = O.batch64(q.detach(), k.detach(), v.detach(), H, Hk, D, spans, left, right, sinks, q_start, keymask.reshape(-1) if keymask is not None else None, scale, do, mult, dtype)
    O.check(o.detach(), want["o"], "o")
    if grad:
        got = torch.autograd.grad(o, (q, k, v), do)
        for n, g in zip(("dq", "dk", "dv"), got):
            O.check(g, want[n], n)
    return o


SQUARE = [  # nseq, L, H, Hk, D, window, sinks, mask
    (1, 1, 1, 1, 64, (0, 0), 0, None),
    (2, 2, 2, 1, 32, (1, 0), 1, None),
    (3, 31, 4, 2, 64, (5, 3), 2, None),
    (1, 32, 3, 3, 128, (-1, 0), 0, None),
    (2, 33, 2, 2, 64, (0, 40), 0, "pad"),
    (3, 65, 6, 2, 64, (16, 16), 4, "holes"),
    (1, 127, 2, 1, 32, (-1, -1), 0, None),
    (2, 128, 3, 1, 64, (32, 0), 1, "pad"),
    (1, 129, 2, 2, 128, (64, 64), 33, None),
    (2, 200, 4, 4, 64, (20, 10), 70, "holes"),
    (2, 257, 2, 2, 32, (3, 2), 500, None),              # more sinks than keys
    (3, 320, 2, 1, 64, (10, 5), 0, "front"),            # rows that see nothing
    (1, 577, 8, 8, 32, (100, 100), 3, None),
    (2, 700, 4, 2, 64, (63, 0), 5, None),
    (1, 1300, 2, 1, 128, (200, 0), 4, "holes"),
    (1, 1111, 8, 1, 64, (1, 1), 40, None),              # two sink blocks, eight heads on one
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nseq,L,H,Hk,D,window,sinks,mask", SQUARE)
def test_window_attention_padded_batches(nseq, L, H, Hk, D, window, sinks, mask, dtype):
    run_case(dtype, nseq, L, L, H, Hk, D, window, sinks, mask=mask, seed=L)


ROWS = [  # nseq, Lq, Lk, H, Hk, D, window, sinks, q_start, mask
    (1, 1, 1, 1, 1, 64, (0, 0), 0, 0, None),
    (8, 1, 512, 12, 12, 64, (128, 128), 1, 0, "pad"),
    (2, 1, 777, 8, 2, 128, (-1, 0), 0, 776, None),
    (1, 1, 5000, 4, 1, 64, (-1, 0), 0, 4999, None),     # the key axis split over workgroups
    (3, 1, 3001, 6, 3, 32, (1000, 0), 4, 3000, "holes"),
    (1, 7, 4096, 4, 1, 64, (-1, -1), 0, 2000, None),    # 28 rows of one block
    (2, 5, 900, 6, 1, 128, (300, 2), 2, 895, "pad"),
    (1, 1, 2049, 32, 1, 64, (-1, 0), 0, 2048, None),    # 32 heads on one
    (1, 33, 3000, 1, 1, 64, (-1, 0), 0, 2960, None),    # too many rows for one block: the tiled kernel, split
    (1, 70, 2500, 2, 1, 128, (-1, -1), 0, 100, "holes"),
    (2, 40, 100, 3, 3, 32, (9, 9), 3, 50, None),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nseq,Lq,Lk,H,Hk,D,window,sinks,q_start,mask", ROWS)
def test_window_attention_query_rows_against_a_longer_key_axis(nseq, Lq, Lk, H, Hk, D, window, sinks, q_start, mask, dtype):
    run_case(dtype, nseq, Lq, Lk, H, Hk, D, window, sinks, q_start=q_start, mask=mask, seed=Lk)


PACKED = [  # lengths, first, tail, H, Hk, D, window, sinks
    ([1], 0, 0, 2, 2, 64, (4, 4), 1),
    ([5, 0, 1, 64, 33, 130, 2], 0, 0, 4, 2, 64, (20, 10), 2),
    ([300, 7, 129], 3, 40, 2, 1, 32, (-1, 0), 0),       # rows in front of and behind the sequences
    ([0, 0, 257], 0, 1, 3, 3, 128, (40, 0), 5),
    ([700, 1, 600], 0, 0, 2, 1, 64, (50, 50), 36),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths,first,tail,H,Hk,D,window,sinks", PACKED)
def test_window_attention_packed_sequences(lengths, first, tail, H, Hk, D, window, sinks, dtype):
    run_case(dtype, None, None, None, H, Hk, D, window, sinks, lengths=lengths, first=first, tail=tail, seed=sum(lengths))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("mask,drop", [("holes", None), ("front", None), (None, (0.2, 77)), ("holes", (0.1, 99))])
def test_window_attention_packed_sequences_with_mask_and_dropout(mask, drop, dtype):
    run_case(dtype, None, None, None, 4, 2, 64, (20, 10), 3, lengths=[5, 0, 70, 1, 200], first=1, tail=3, mask=mask, drop=drop, seed=3)


def test_window_attention_many_short_sequences():
    """More sequences than a grid's z axis has room for."""
    n = 70000
    q, k, v, g = (rnd((n * 3, 32), BF16, 60 + i) for i in range(4))
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    o = Fn.window_attention(q, k, v, 1, 32, nseq=n, window=(0, 0), sinks=1)
    got = torch.autograd.grad(o, (q, k, v), g)
    at = slice(3 * (n - 5), 3 * n)        # the last five, by themselves
    q2, k2, v2 = (t.detach()[at].clone().requires_grad_(True) for t in (q, k, v))
    o2 = Fn.window_attention(q2, k2, v2, 1, 32, nseq=5, window=(0, 0), sinks=1)
    spans = [(3 * b, 3, 3 * b, 3) for b in range(5)]
    want = O.batch64(q2.detach(), k2.detach(), v2.detach(), 1, 1, 32, spans, 0, 0, 1, 0, None, 32 ** -0.5, g[at], dtype=BF16)
    O.check(o.detach()[at], want["o"], "o")
    O.check(o2.detach(), want["o"], "o of the five")
    for name, x in zip(("dq", "dk", "dv"), got):
        O.check(x[at], want[name], name)


@pytest.mark.parametrize("Lq", [1, 200])
def test_window_attention_offsets_beyond_32_bits(Lq):
    """Key rows 4 KB apart, 1.1 million of them: the last window lies 4.5 GB behind the sinks."""
    Lk, H, D, left, sinks = 1100000, 2, 64, 90, 4
    buf = torch.zeros((Lk, 2048), dtype=BF16, device=DEV)
    near = torch.cat([torch.arange(sinks), torch.arange(Lk - Lq - left, Lk)]).to(DEV)
    buf[near, :2 * H * D] = rnd((len(near), 2 * H * D), BF16, 5)
    k, v = buf[:, :H * D].requires_grad_(True), buf[:, H * D:2 * H * D].requires_grad_(True)
    q = rnd((Lq, H * D), BF16, 6).requires_grad_(True)
    g = rnd((Lq, H * D), BF16, 7)
    o = Fn.window_attention(q, k, v, H, D, window=(left, 0), sinks=sinks, q_start=Lk - Lq)
    got = torch.autograd.grad(o, (q, k, v), g)
    # the same rows without what lies between: positions shift, the sinks stay in front of every window
    n = len(near)
    want = O.batch64(q.detach(), k.detach()[near], v.detach()[near], H, H, D, [(0, Lq, 0, n)], left, 0, sinks, n - Lq, None, D ** -0.5, g, dtype=BF16)
    O.check(o.detach(), want["o"], "o")
    O.check(got[0], want["dq"], "dq")
    for name, x in zip(("dk", "dv"), got[1:]):
        O.check(x[near], want[name], name)
        assert not x[sinks:Lk - Lq - left].any()


def test_window_attention_on_two_streams_at_once():
    """Calls that split the key axis, running at the same time on two streams, have a workspace each."""
    q, k, v = rnd((1, 256), BF16, 1), rnd((20000, 256), BF16, 2), rnd((20000, 256), BF16, 3)
    calls = [dict(window=(-1, 0), q_start=19999), dict(window=(9000, 0), q_start=12000)]
    want = [Fn.window_attention(q, k, v, 4, 64, **c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(5):
        for i, (st, c) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(st):
                got[i].append(Fn.window_attention(q, k, v, 4, 64, **c))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_the_backend_refuses_tensors_of_the_cpu():
    with pytest.raises(TypeError, match="on the GPU"):
        Fn.window_attention(torch.zeros(4, 64), torch.zeros(4, 64), torch.zeros(4, 64), 1, 64)
    with pytest.raises(TypeError, match="on the GPU"):
        Fn.rotary(torch.zeros(4, 64), None, Fn.RotaryPositions(64), 64)


def test_no_derivative_of_the_gradient():
    q = rnd((8, 64), F32, 1).requires_grad_(True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(Fn.window_attention(q, q, q, 1, 64, window=2).sum(), q, create_graph=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nseq,Lq,Lk,H,Hk,D,window,sinks,q_start", [(2, 150, 150, 4, 2, 64, (30, 30), 2, 0), (2, 1, 150, 4, 4, 32, (40, 0), 1, 0), (1, 97, 97, 2, 1, 128, (-1, 0), 0, 0),
                                                                   (1, 600, 600, 2, 2, 64, (7, 0), 35, 0)])
def test_window_attention_dropout(nseq, Lq, Lk, H, Hk, D, window, sinks, q_start, dtype):
    run_case(dtype, nseq, Lq, Lk, H, Hk, D, window, sinks, q_start=q_start, drop=(0.25, 1234567), seed=Lq + 1)


def test_window_attention_gradient_against_differences():
    L, H, D = 70, 2, 32
    q, k, v = (rnd((L, H * D), F32, 20 + i, 0.7).requires_grad_(True) for i in range(3))
    g = rnd((L, H * D), F32, 30)
    dirs = [rnd((L, H * D), F32, 40 + i) for i in range(3)]

    def f(t):      # in 64 bits from the 64-bit form at shifted inputs; the kernel's gradient is what is tested
        r = O.batch64(q.detach().double() + t * dirs[0], k.detach().double() + t * dirs[1], v.detach().double() + t * dirs[2], H, H, D, [(0, L, 0, L)], 12, 5, 3, 0, None,
                      1 / math.sqrt(D))
        return (r["o"][0] * g.double()).sum()
    h = 1e-4
    num = (f(h) - f(-h)) / (2 * h)
    got = torch.autograd.grad(Fn.window_attention(q, k, v, H, D, window=(12, 5), sinks=3), (q, k, v), g)
    dot = sum((a.double() * d.double()).sum() for a, d in zip(got, dirs))
    want = O.batch64(q.detach(), k.detach(), v.detach(), H, H, D, [(0, L, 0, L)], 12, 5, 3, 0, None, 1 / math.sqrt(D), g)
    room = sum((want[n][1] * d.abs().double()).sum() for n, d in zip(("dq", "dk", "dv"), dirs)) + 1e-6 * num.abs()      # h^2 f''' of the difference
    assert abs(dot - num) <= room


def test_window_attention_broadcast_inputs_and_other_streams():
    """Expanded inputs (row stride 0) get the sum of their rows' gradients; a call on another stream gives the same bits."""
    L, H, D = 100, 2, 64
    one = rnd((1, H * D), BF16, 3).requires_grad_(True)
    k, v = rnd((L, H * D), BF16, 4), rnd((L, H * D), BF16, 5)
    g = rnd((L, H * D), BF16, 6)
    (dq,) = torch.autograd.grad(Fn.window_attention(one.expand(L, H * D), k, v, H, D, window=8), one, g)
    full = one.detach().expand(L, H * D).contiguous().requires_grad_(True)
    (dfull,) = torch.autograd.grad(Fn.window_attention(full, k, v, H, D, window=8), full, g)
    assert torch.equal(dq, dfull.sum(0, keepdim=True))
    want = Fn.window_attention(full.detach(), k, v, H, D, window=8)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = Fn.window_attention(full.detach(), k, v, H, D, window=8)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got, want)


def test_every_result_is_reproducible():
    """Split key axes, sinks and shared heads: a second run gives the same bits."""
    for kw in (dict(nseq=1, Lq=1, Lk=6000, H=8, Hk=2, D=64, window=(-1, 0), q_start=5999), dict(nseq=2, Lq=900, Lk=900, H=4, Hk=1, D=64, window=(100, 0), q_start=0)):
        q, k, v = rnd((kw["nseq"] * kw["Lq"], kw["H"] * kw["D"]), BF16, 1), rnd((kw["nseq"] * kw["Lk"], kw["Hk"] * kw["D"]), BF16, 2), rnd((kw["nseq"] * kw["Lk"], kw["Hk"] * kw["D"]), BF16, 3)
        q, k, v = (t.requires_grad_(True) for t in (q, k, v))
        g = rnd(tuple(q.shape), BF16, 4)
        runs = []
        for _ in range(2):
            o = Fn.window_attention(q, k, v, kw["H"], kw["D"], nseq=kw["nseq"], kv_heads=kw["Hk"], window=kw["window"], sinks=4, q_start=kw["q_start"])
            runs.append([o.detach(), *torch.autograd.grad(o, (q, k, v), g)])
        assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_captured_and_replayed_with_a_workspace_each():
    """Two graphs whose calls split the key axis, replayed alternately with other inputs between: each replay equals the eager result."""
    H, D, L = 4, 64, 5000
    q, k, v = rnd((1, H * D), BF16, 1), rnd((L, H * D), BF16, 2), rnd((L, H * D), BF16, 3)
    rope = Fn.RotaryPositions(64)

    def step(window):
        return Fn.window_attention(Fn.rotary(q, None, rope, D, start=L - 1), Fn.rotary(k, None, rope, D), v, H, D, window=window, q_start=L - 1)
    for w in ((-1, 0), (4000, 0)):
        step(w)
    graphs, outs = [], []
    for w in ((-1, 0), (4000, 0)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(w))
        graphs.append(g)
    for rep in range(3):
        for t in (q, k, v):
            t.copy_(rnd(tuple(t.shape), BF16, 50 + rep))
        want = [step((-1, 0)), step((4000, 0))]
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


SPLIT = [  # nseq, Lq, Lk, H, Hk, D, window, sinks, q_start, mask, dropout: passes split over workgroups in many parts, in few, of many rows
    (1, 1000, 1000, 8, 2, 64, (-1, -1), 0, 0, None, None),      # more than eight parts of every key
    (1, 900, 900, 2, 1, 128, (-1, 0), 3, 0, "pad", None),
    (1, 1030, 1030, 4, 4, 128, (200, 100), 40, 0, "holes", (0.1, 5)),     # two waves to a key block, two sink blocks
    (2, 300, 300, 4, 2, 128, (30, 0), 2, 0, "front", (0.2, 6)),
    (1, 2048, 2048, 3, 3, 32, (256, 256), 1, 0, None, None),    # two to eight parts, and the sinks' chunks
    (1, 200, 2000, 6, 3, 64, (-1, 0), 0, 1800, "holes", None),
    (1, 200, 2000, 24, 24, 32, (1500, 0), 5, 1700, None, (0.3, 7)),       # more than 4096 rows and heads to join
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("nseq,Lq,Lk,H,Hk,D,window,sinks,q_start,mask,drop", SPLIT)
def test_window_attention_split_passes(nseq, Lq, Lk, H, Hk, D, window, sinks, q_start, mask, drop, dtype):
    run_case(dtype, nseq, Lq, Lk, H, Hk, D, window, sinks, q_start=q_start, mask=mask, drop=drop, seed=Lk + D)


@pytest.mark.parametrize("L,H,D,window,sinks", [(300, 4, 64, (8, 2), 1), (20, 4, 64, (-1, -1), 0), (7, 2, 32, (-1, 0), 0), (300, 2, 128, (16, 0), 1)])
def test_few_visible_keys_in_training_cost_one_rounding(L, H, D, window, sinks):
    """Up to 64 visible keys the probabilities' rounding does not reach the output that the backward pass builds on: half a step of the output, and next to it what f32 scores
    (D products of a sum of about 5 in magnitude, the row's sum once more: 2 * 64 * 5 * 2^-24 < 2^-14) and twice rounded probabilities (2^-17) leave, of sum P |v|."""
    q, k, v = (rnd((L, H * D), BF16, 90 + i) for i in range(3))
    o = Fn.window_attention(q.requires_grad_(True), k, v, H, D, window=window, sinks=sinks).detach().double()
    exact, room = (O.batch64(q.detach(), k, x, H, H, D, [(0, L, 0, L)], *window, sinks, 0, None, 1 / math.sqrt(D), None, None, BF16)["o"][0] for x in (v, v.abs()))
    assert ((o - exact.to(o)).abs() <= 2.0 ** -8 * exact.abs().to(o) + 2.0 ** -14 * room.to(o)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window,sinks,D", [((-1, -1), 0, 64), ((40, 10), 3, 64), ((30, 0), 2, 128)])
def test_mask_that_drowns_the_scores(window, sinks, D, dtype):
    """-1e9 on every key of a sequence: the scores are below the mask's last bit, so every visible key counts the same, in the gradients as in the output."""
    L, H = 150, 2
    q, k, v, do = (rnd((L, H * D), dtype, 70 + i) for i in range(4))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = Fn.window_attention(*leaves, H, D, window=window, sinks=sinks, keymask=torch.full((L,), -1e9, device=DEV))
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    i, j = torch.arange(L)[:, None], torch.arange(L)[None, :]
    left, right = (L if x < 0 else x for x in window)
    see = (j <= i + right) & ((j >= i - left) | (j < sinks))
    P = see.double() / see.sum(1, keepdim=True)
    q, k, v, do = (t.detach().double().cpu().view(L, H, D).transpose(0, 1) for t in (q, k, v, do))
    dP = do @ v.transpose(1, 2)
    dS = P * (dP - (P * dP).sum(2, keepdim=True)) / math.sqrt(D)
    half = torch.finfo(dtype).eps / 2
    # roundings: P, dS to the operand type, the result, and the row sums under dS (two terms of P |dP|); f32 sums of up to L terms
    sums = L * O.U32
    room_S = P * (dP.abs() + 2 * (P * dP.abs()).sum(2, keepdim=True)) / math.sqrt(D)
    for got, want, room in ((o, P @ v, P @ v.abs()), (dv, P.t() @ do, P.t() @ do.abs()), (dq, dS @ k, room_S @ k.abs()), (dk, dS.transpose(1, 2) @ q, room_S.transpose(1, 2) @ q.abs())):
        got = got.detach().double().cpu().view(L, H, D).transpose(0, 1)
        assert ((got - want).abs() <= half * want.abs() + (half + 4 * sums) * room).all()


@pytest.mark.parametrize("dtype,pitch", [(BF16, 5 * 2 ** 20), (F32, 3 * 2 ** 20 + 64)])
def test_rows_far_apart(dtype, pitch):
    """The [CLS] rows of long sequences inside their projection: more than 8 MB between two rows of q, and between the rows of its gradient."""
    H, D, Lk, n = 2, 64, 300, 3
    buf = torch.zeros((n, pitch), dtype=dtype, device=DEV)
    buf[:, :H * D] = rnd((n, H * D), dtype, 1)
    q = buf[:, :H * D].detach().requires_grad_(True)
    k, v, do = rnd((n * Lk, H * D), dtype, 2).requires_grad_(True), rnd((n * Lk, H * D), dtype, 3).requires_grad_(True), rnd((n, H * D), dtype, 4)
    assert q.stride(0) == pitch
    wide = torch.zeros_like(buf)
    wide[:, :H * D] = do
    o = Fn.window_attention(q, k, v, H, D, nseq=n, window=(50, 50), sinks=1)
    want = O.batch64(q.detach(), k.detach(), v.detach(), H, H, D, [(b, 1, b * Lk, Lk) for b in range(n)], 50, 50, 1, 0, None, D ** -0.5, do, None, dtype)
    O.check(o.detach(), want["o"], "o")
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), wide[:, :H * D])):
        O.check(g, want[name], name)


def test_positions_changed_before_the_backward_pass_are_refused():
    x = rnd((40, 64), F32, 1).requires_grad_(True)
    positions = torch.arange(40, device=DEV)
    y = Fn.rotary(x, None, Fn.RotaryPositions(64), 64, positions=positions)
    positions.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@pytest.mark.parametrize("L,H,D,window,sinks", [(4, 4, 64, (10, 0), 0), (100, 2, 64, (20, 5), 3), (70, 2, 32, (-1, -1), 0), (90, 2, 128, (30, 0), 2)])
def test_small_gradients_cost_one_rounding(L, H, D, window, sinks):
    """Where few pairs are visible P and dS enter the products to 2^-17: half a step of each gradient, and next to it of the sums of absolute terms what f32 scores (2^-14, see above),
    the remainders (2^-17 each) and f32 sums (D, L and the row sums: 3 * 128 * 2^-24 < 2^-15) leave: less than 2^-13."""
    q, k, v, do = (rnd((L, H * D), BF16, 80 + i) for i in range(4))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(Fn.window_attention(*leaves, H, D, window=window, sinks=sinks), leaves, do)
    i, j = torch.arange(L)[:, None], torch.arange(L)[None, :]
    left, right = (L if x < 0 else x for x in window)
    see = (j <= i + right) & ((j >= i - left) | (j < sinks))
    q, k, v, do = (t.detach().double().cpu().view(L, H, D).transpose(0, 1) for t in (q, k, v, do))
    P = ((q @ k.transpose(1, 2)) / math.sqrt(D)).masked_fill(~see, -math.inf).softmax(2)
    dP, dP_abs = do @ v.transpose(1, 2), do.abs() @ v.abs().transpose(1, 2)
    dS = P * (dP - (P * dP).sum(2, keepdim=True)) / math.sqrt(D)
    room = P * (dP_abs + (P * dP_abs).sum(2, keepdim=True)) / math.sqrt(D)
    for g, want, r in zip(got, (dS @ k, dS.transpose(1, 2) @ q, P.transpose(1, 2) @ do), (room @ k.abs(), room.transpose(1, 2) @ q.abs(), P.transpose(1, 2) @ do.abs())):
        g = g.double().cpu().view(L, H, D).transpose(0, 1)
        assert ((g - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -13 * r).all()


def test_training_captured_and_replayed():
    """Forward and backward of both operators in one graph, with sinks' and split keys' partial sums: each replay equals the eager result."""
    H, D, L = 2, 64, 1500
    q, k, v, g = (rnd((L, H * D), BF16, i) for i in range(4))
    rope = Fn.RotaryPositions(64)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        a, b = Fn.rotary(leaves[0], leaves[1], rope, D, start=7)
        o = Fn.window_attention(a, b, leaves[2], H, D, window=(300, 20), sinks=3)
        return [o.detach(), *torch.autograd.grad(o, leaves, g)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(3):
        for i, t in enumerate((q, k, v, g)):
            t.copy_(rnd(tuple(t.shape), BF16, 60 + 4 * rep + i))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


# ------------------------------------------------------------------------------------------------- the operators together

@pytest.mark.parametrize("cls_only", [False, True])
@pytest.mark.parametrize("options", O.BERT_OPTIONS)
def test_text_tower_with_long_report_options(options, cls_only):
    """Two layers in f32: ten products of at most 130 terms each way, sums of magnitudes some three times the values: 10 * 130 * 3 * 2^-24 = 2.3e-4 at worst, of either sign."""
    T = 30 if options.get("position_embedding_type") != "rotary" else 150
    got, want, grads, rotary = O.bert_case(options, T, DEV, cls_only=cls_only)
    assert (got.double() - want).abs().max() <= 2e-4 * want.abs().max()
    for n, (a, b) in grads.items():
        if "pooler" in n or (rotary and "position_embeddings" in n):
            assert a is None
            continue
        assert (a.double() - b).norm() <= 4e-4 * b.norm() + 1e-6, n


@pytest.mark.parametrize("options", O.BERT_OPTIONS)
def test_text_tower_with_long_report_options_mixed_precision(options):
    """f32 stream, bf16 matrix operands: in each of two layers seven roundings (2^-8 at most each) stand between the input and the output, and twice that in the gradients;
    a key bias shifts every score of a row alike, so its true gradient is zero and what is left is held to the query bias's scale."""
    T = 30 if options.get("position_embedding_type") != "rotary" else 150
    got, want, grads, rotary = O.bert_case(options, T, DEV, operand_dtype=BF16)
    assert (got.double() - want).norm() <= 14 * 2.0 ** -8 * want.norm()
    for n, (a, b) in grads.items():
        if "pooler" in n or (rotary and "position_embeddings" in n):
            assert a is None
            continue
        scale = grads[n.replace("self.key", "self.query")][1].norm() if "key.bias" in n else b.norm()
        assert (a.double() - b).norm() <= 28 * 2.0 ** -8 * scale, n


def test_text_tower_cls_rows_of_a_long_batch():
    """BERT-base's width at 2000 tokens: the [CLS] rows lie 9 MB apart inside the projection.  The same rows as from the pass over every token, up to bf16 (two roundings of the
    layer's attention output, each half a step, through layers of norm about 1)."""
    from transformers import BertConfig, BertModel
    from ct_clip_amd.bert import bert_last_hidden_state
    torch.manual_seed(0)
    cfg = BertConfig(vocab_size=50, hidden_size=768, num_hidden_layers=1, num_attention_heads=12, intermediate_size=768, position_embedding_type="rotary", attention_window=64,
                     attention_sinks=1, hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0)
    bert = BertModel(cfg, add_pooling_layer=False).to(DEV)
    ids = torch.randint(0, 50, (2, 2000), device=DEV)
    mask = (torch.arange(2000, device=DEV)[None, :] < torch.tensor([[2000], [1500]], device=DEV)).long()
    every = bert_last_hidden_state(bert, ids, mask, BF16).view(2, 2000, 768)[:, 0]
    rows = bert_last_hidden_state(bert, ids, mask, BF16, cls_only=True)
    assert rows.shape == (2, 768) and torch.isfinite(rows).all()
    assert (rows.float() - every.float()).abs().max() <= 4 * 2.0 ** -8 * every.abs().max().float()
    rows.float().square().sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in bert.parameters() if p.grad is not None)
