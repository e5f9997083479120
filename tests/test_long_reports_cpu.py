"""Rotary positions and windowed attention without a device: frequencies, packed tables, what is refused (by the functions and at the C entries), and the host
composition -- autograd nodes and the text tower -- on a torch backend against the 64-bit forms."""
import ctypes
import math

import numpy as np
import pytest
import torch

from ct_clip_amd import backend
from ct_clip_amd import functional as Fn
from tests import long_report_oracle as O
from tests.ref_backend import RefBackend


class RefOps(RefBackend):
    """The two operators in plain torch, 64 bits inside, with the interface of the HIP backend."""

    def rotary(self, q, k, turns, D, rot, L, positions, start, interleaved, magnitude, inverse=False, out=None):
        freq = torch.tensor([(int(t) % 2 ** 64) * 2.0 ** -64 for t in turns], dtype=torch.float64) * 2 * math.pi
        pos = positions if positions is not None else start + torch.arange(q.shape[0]) % L
        new = [None if t is None else O.rotary64(t, freq, magnitude, D, rot, interleaved, pos, inverse)[0].to(t.dtype) for t in (q, k)]
        if out is None:
            return tuple(new)
        for o, n in zip(out, new):
            if o is not None:
                o.copy_(n)
        return out

    @staticmethod
    def _spans(geo):
        if geo.packed:
            e = geo.tables(torch.device("cpu"))[0].tolist()
            return [(a, b - a, a, b - a) for a, b in zip(e, e[1:])]
        return [(b * geo.Lq, geo.Lq, b * geo.Lk, geo.Lk) for b in range(geo.nseq)]

    def _run(self, q, k, v, keymask, geo, scale, dropout, dout=None):
        drop = self.attn_dropout_mask(geo.nseq, geo.H, geo.Lk, dropout[0], dropout[1], q.device) if dropout else None
        return O.batch64(q.detach(), k.detach(), v.detach(), geo.H, geo.Hk, geo.D, self._spans(geo), geo.left, geo.right, geo.sinks, geo.q_start, keymask, scale, dout, drop)

    def win_attn_fwd(self, q, k, v, keymask, geo, scale, want_lse=True, dropout=None):
        keymask = keymask.reshape(-1) if keymask is not None else None
        return self._run(q, k, v, keymask, geo, scale, dropout)["o"][0].to(q.dtype), torch.zeros(geo.H, geo.Mq) if want_lse else None, None

    def win_attn_bwd(self, q, k, v, keymask, geo, scale, o, dout, lse, o_lo=None, dropout=None, out=None):
        r = self._run(q, k, v, keymask.reshape(-1) if keymask is not None else None, geo, scale, dropout, dout)
        new = [r[n][0].to(q.dtype) for n in ("dq", "dk", "dv")]
        if out is None:
            return tuple(new)
        for t, n in zip(out, new):
            t.copy_(n)
        return out


@pytest.fixture
def ref():
    prev = backend.use(RefOps())
    yield
    backend.use(prev)


# --------------------------------------------------------------------------------------------------------------------- plans

def test_frequencies():
    r = Fn.RotaryPositions(64)
    want = 10000.0 ** (-np.arange(32) / 32)
    np.testing.assert_allclose(r.frequencies, want, rtol=1e-14)
    np.testing.assert_allclose([int(b) * 2.0 ** -64 * 2 * math.pi for b in r.bits], want, rtol=1e-14)
    assert r.magnitude == 1.0
    np.testing.assert_allclose(Fn.RotaryPositions(64, scaling=dict(type="linear", factor=4)).frequencies, want / 4, rtol=1e-14)
    n = Fn.RotaryPositions(64, scaling=dict(type="ntk", factor=4)).frequencies
    np.testing.assert_allclose(n[-1], want[-1] / 4, rtol=1e-12)          # the slowest pair is stretched by the whole factor, the first not at all
    assert n[0] == 1.0
    y = Fn.RotaryPositions(64, scaling=dict(type="yarn", factor=8, original_length=512))
    assert y.frequencies[0] == want[0] and abs(y.frequencies[-1] / want[-1] - 1 / 8) < 1e-12 and abs(y.magnitude - (0.1 * math.log(8) + 1)) < 1e-15
    assert np.all(np.diff(y.frequencies) < 0)
    assert Fn.RotaryPositions(64, scaling=dict(type="yarn", factor=8, original_length=512, attention_factor=2.0)).magnitude == 2.0
    t = r.turns(torch.device("cpu"))
    assert t.dtype == torch.int64 and [int(x) % 2 ** 64 for x in t] == [int(b) for b in r.bits] and r.turns(torch.device("cpu")) is t


@pytest.mark.parametrize("args,kw", [((3,), {}), ((0,), {}), ((64,), dict(layout="pairs")), ((64,), dict(base=1.0)), ((64,), dict(base=math.inf)),
                                     ((64,), dict(scaling=dict(type="cubic", factor=2))), ((64,), dict(scaling=dict(type="linear", factor=0.5))),
                                     ((64,), dict(scaling=dict(type="yarn", factor=2))), ((64,), dict(scaling=dict(type="linear", factor=2, extra=1))),
                                     ((64,), dict(scaling=dict(type="yarn", factor=2, original_length=512, beta_fast=1, beta_slow=32)))])
def test_rotary_plan_refuses(args, kw):
    with pytest.raises(ValueError):
        Fn.RotaryPositions(*args, **kw)


def test_packed_sequences():
    s = Fn.PackedSequences([300, 0, 1, 128], first=2)
    off, tiles = s.on(torch.device("cpu"))
    assert off.tolist() == [2, 302, 302, 303, 431] and tiles.reshape(-1, 2).tolist() == [[0, 0], [0, 1], [0, 2], [2, 0], [3, 0]]
    assert (s.rows, s.end, s.longest, s.ntiles) == (429, 431, 300, 5) and off.dtype == tiles.dtype == torch.int32
    for bad in (dict(lengths=[1, -1]), dict(lengths=[1], first=-1), dict(lengths=[2 ** 31])):
        with pytest.raises(ValueError):
            Fn.PackedSequences(**bad)


# ------------------------------------------------------------------------------------------------------------------ refusals

def test_functions_refuse(ref):
    rope, x = Fn.RotaryPositions(32), torch.zeros(6, 64)
    for call in (lambda: Fn.rotary(x, None, rope, 24), lambda: Fn.rotary(x, x[:5], rope, 32), lambda: Fn.rotary(x, x.bfloat16(), rope, 32), lambda: Fn.rotary(x, None, rope, 16),
                 lambda: Fn.rotary(x, None, rope, 32, L=0), lambda: Fn.rotary(x, None, rope, 32, positions=torch.zeros(6)), lambda: Fn.rotary(x, None, rope, 32, start=2 ** 63),
                 lambda: Fn.rotary(x, None, rope, 32, positions=torch.zeros(5, dtype=torch.int64)), lambda: Fn.rotary(x[0], None, rope, 32)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        Fn.rotary(x, None, 10000.0, 32)
    q, k = torch.zeros(6, 128), torch.zeros(6, 64)
    ok = dict(kv_heads=1, window=3)
    Fn.window_attention(q, k, k, 2, 64, **ok)
    for kw in (dict(ok, kv_heads=2), dict(ok, window=(-2, 0)), dict(ok, sinks=-1), dict(ok, q_start=1), dict(ok, nseq=4), dict(ok, nseq=0), dict(ok, scale=0.0), dict(ok, scale=-1.0),
               dict(ok, scale=math.inf), dict(ok, keymask=torch.zeros(5)), dict(ok, keymask=torch.zeros(6, dtype=torch.int64)), dict(ok, dropout=(1.0, 1)), dict(ok, dropout=(-0.1, 1)),
               dict(ok, nseq=Fn.PackedSequences([7])), dict(ok, nseq=Fn.PackedSequences([6], first=1)), dict(ok, nseq=Fn.PackedSequences([3]), q_start=1)):
        with pytest.raises(ValueError):
            Fn.window_attention(q, k, k, 2, 64, **kw)
    for a in ((q, k, k[:5], 2, 64), (q, k, k, 3, 64), (q, k, k.bfloat16(), 2, 64), (q, k, k, 1, 128)):
        with pytest.raises(ValueError):
            Fn.window_attention(*a, **ok)
    with pytest.raises(ValueError, match="32, 64 or 128"):
        Fn.window_attention(torch.zeros(6, 96), torch.zeros(6, 48), torch.zeros(6, 48), 2, 48, kv_heads=1)
    with pytest.raises(TypeError):
        Fn.window_attention(q.half(), k.half(), k.half(), 2, 64, **ok)
    with pytest.raises(ValueError):          # more query rows than keys
        Fn.window_attention(q, k[:3], k[:3], 2, 64, **ok)


def test_c_entries_answer_before_any_launch():
    from ct_clip_amd import _lib
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def rot(q=p, k=p, qo=p, ko=p, turns=p, pos=None, pb=0, M=4, L=4, Hq=2, Hk=2, D=64, r=64, ldq=128, ldk=128, ldqo=128, ldko=128, dt=1):
        return lib.ctclip_rotary(q, k, qo, ko, turns, pos, pb, M, L, 0, Hq, Hk, D, r, ldq, ldk, ldqo, ldko, 0, 1.0, 0, dt, None)
    assert rot(q=None) == rot(turns=None) == rot(k=None) == rot(qo=None) == -1
    assert rot(r=66) == rot(r=3) == rot(r=0) == rot(M=-1) == rot(L=0) == rot(Hq=0) == rot(pos=p, pb=2) == rot(ldqo=100) == -1
    assert rot(qo=p + 256) == rot(ldqo=256) == -1            # one tensor in place and the other not; in place with another pitch
    assert rot(dt=2) == -2
    assert rot(M=0, q=None) == 0 and lib.ctclip_last_error()

    def fwd(q=p, k=p, v=p, off=None, tiles=None, nt=0, out=p, nseq=2, Lq=8, Lk=8, Mq=16, Mk=16, H=2, Hk=1, D=64, left=4, right=4, sinks=1, q0=0, ldq=128, ldk=64, ldv=64, ldo=128,
            scale=1.0, drop=0.0, dt=1, ws=None, n=0):
        return lib.ctclip_win_attn_fwd(q, k, v, None, off, tiles, nt, out, None, None, nseq, Lq, Lk, Mq, Mk, H, Hk, D, left, right, sinks, q0, ldq, ldk, ldv, ldo, scale, drop, 0, dt, ws, n, None)
    assert fwd(q=None) == fwd(k=None) == fwd(v=None) == fwd(out=None) == fwd(q=p + 2) == fwd(ldk=65) == fwd(ldo=120) == -1
    assert fwd(H=3, Hk=2) == fwd(left=-2) == fwd(sinks=-1) == fwd(q0=1) == fwd(Mq=17) == fwd(Lq=9, Mq=18) == fwd(scale=0.0) == fwd(scale=-1.0) == fwd(drop=1.0) == -1
    assert fwd(scale=math.nan) == fwd(drop=math.nan) == fwd(off=p, Mq=16, nt=2) == fwd(off=p, tiles=p, nt=2, Mk=15) == -1
    assert fwd(D=48) == fwd(dt=2) == -2
    assert fwd(nseq=1, Lq=1, Lk=5000, Mq=1, Mk=5000, left=-1, q0=4999) == -3 and b"workspace" in lib.ctclip_last_error()
    assert fwd(nseq=0, Mq=0, Mk=0) == fwd(Lq=0, Mq=0) == fwd(off=p, nt=0) == 0

    def bwd(q=p, lse=p, delta=p, dq=p, ldq=128, lddq=128, nseq=2, L=8, left=4, sinks=0, ws=None, n=0, dt=1, D=64, scale=1.0):
        M = nseq * L
        return lib.ctclip_win_attn_bwd(q, p, p, None, None, None, 0, p, None, p, lse, delta, dq, p, p, nseq, L, L, M, M, 2, 1, D, left, 0, sinks, 0, ldq, 64, 64, 128, 128, lddq, 64, 64,
                                       scale, 0.0, 0, dt, ws, n, None)
    assert bwd(q=None) == bwd(lse=None) == bwd(delta=None) == bwd(dq=None) == bwd(dq=p + 8) == bwd(lddq=64) == bwd(scale=0.0) == -1
    assert bwd(D=96) == bwd(dt=3) == -2
    assert bwd(L=64, sinks=2) == -3 and bwd(nseq=0) == 0
    assert lib.ctclip_win_attn_fwd_workspace(1, 8, 8, 2, 1, 64, 4, 4, 1, 0, 0) == 0 and lib.ctclip_win_attn_fwd_workspace(1, 1, 5000, 2, 1, 64, -1, 0, 0, 4999, 0) > 0
    assert lib.ctclip_win_attn_bwd_workspace(0, 8, 8, 0, 2, 1, 64, 4, 4, 1, 0, 0) == 0 and lib.ctclip_win_attn_bwd_workspace(1, 64, 64, 64, 2, 1, 64, 4, 4, 1, 0, 0) > 0


def test_c_entries_refuse_rows_that_a_launch_cannot_reach():
    from ct_clip_amd import _lib
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def fwd(ldq=64, ldk=64, L=128):
        return lib.ctclip_win_attn_fwd(p, p, p, None, None, None, 0, p, None, None, 1, L, L, L, L, 1, 1, 64, 4, 4, 0, 0, ldq, ldk, 64, 64, 1.0, 0.0, 0, 1, None, 0, None)
    assert fwd(ldq=2 ** 24) == fwd(ldk=2 ** 24) == fwd(ldk=2 ** 24, L=70) == -2 and b"2 GiB" in lib.ctclip_last_error()
    assert fwd(ldq=2 ** 31) == fwd(ldk=2 ** 30) == -1
    assert lib.ctclip_rotary(p, None, p, None, p, None, 0, 2 ** 28, 1, 0, 1, 0, 8, 8, 8, 0, 8, 0, 1, 1.0, 0, 1, None) == -2


# --------------------------------------------------------------------------------------------------------------- composition

def test_bounds_notice_a_wrong_oracle():
    """The comparison itself: a key too many in the window, a sink too few, an angle off by one position are all found."""
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(40, 64, generator=g) for _ in range(4))
    span = [(0, 40, 0, 40)]
    good = O.batch64(q, k, v, 2, 2, 32, span, 5, 2, 2, 0, None, 0.2, do)
    for left, right, sinks in ((6, 2, 2), (5, 1, 2), (5, 2, 1)):
        bad = O.batch64(q, k, v, 2, 2, 32, span, left, right, sinks, 0, None, 0.2, do, dtype=torch.bfloat16)
        for n in good:
            O.check(good[n][0], good[n], n)
            with pytest.raises(AssertionError):
                O.check(good[n][0], bad[n], n)
    f, pos = torch.from_numpy(Fn.RotaryPositions(32).frequencies), torch.arange(40)
    y, m = O.rotary64(q, f, 1.0, 32, 32, False, pos)
    with pytest.raises(AssertionError):
        O.check(O.rotary64(q, f, 1.0, 32, 32, False, pos + 1)[0], (y, O.rotary_bound(y, m, torch.bfloat16)), "y")


def test_nodes_pass_gradients_in_the_caller_s_layout(ref):
    """Column views, shared heads, a missing k, an empty call."""
    buf = torch.randn(20, 2 * 64 + 2 * 32, requires_grad=True)
    rope = Fn.RotaryPositions(16, layout="interleaved")
    q, k = Fn.rotary(buf[:, :128], buf[:, 128:160], rope, 32, L=10)
    o = Fn.window_attention(q, k, buf[:, 160:], 4, 32, nseq=2, kv_heads=1, window=(3, 0), sinks=1)
    do = torch.randn(20, 128)
    (got,) = torch.autograd.grad(o, buf, do)
    x = buf.detach().double().requires_grad_(True)
    f, pos = torch.from_numpy(rope.frequencies), torch.arange(20) % 10
    q, k = O.rotary64(x[:, :128], f, 1.0, 32, 16, True, pos)[0], O.rotary64(x[:, 128:160], f, 1.0, 32, 16, True, pos)[0]
    see = O.visible(10, 10, 3, 0, 1, 0)
    outs = []
    for b in range(2):
        at = slice(10 * b, 10 * b + 10)
        Q, K, V = q[at].reshape(10, 4, 32).transpose(0, 1), k[at][None], x[at, 160:][None]
        outs.append((torch.softmax((Q @ K.transpose(1, 2) / math.sqrt(32)).masked_fill(~see, -math.inf), -1) @ V).transpose(0, 1).reshape(10, 128))
    want = torch.autograd.grad(torch.cat(outs), x, do.double())[0]
    # the nodes hand f32 tensors on: three roundings between the 64-bit pieces, 2^-24 each of values of a few units
    torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=2e-6)
    one = Fn.rotary(buf[:, :64], None, rope, 32)
    assert torch.is_tensor(one) and one.requires_grad
    e = torch.zeros(0, 64, requires_grad=True)
    kk = torch.randn(5, 64, requires_grad=True)
    r = Fn.window_attention(e, kk, kk, 2, 32, nseq=1)
    assert r.shape == (0, 64)
    ge, gk = torch.autograd.grad(r.sum(), (e, kk))
    assert ge.shape == (0, 64) and not gk.any()
    none = Fn.window_attention(kk, kk, kk, 2, 32, nseq=Fn.PackedSequences([0, 0]))
    assert not none.any()


@pytest.mark.parametrize("cls_only", [False, True])
@pytest.mark.parametrize("options", O.BERT_OPTIONS)
def test_text_tower_with_long_report_options(ref, options, cls_only):
    T = 30 if options.get("position_embedding_type") != "rotary" else 50          # (rotary: beyond the 32 rows of the position table)
    got, want, grads, rotary = O.bert_case(options, T, "cpu", cls_only=cls_only)
    torch.testing.assert_close(got.double(), want, rtol=2e-5, atol=2e-5)          # two layers in f32: ~30 roundings of values of order 1
    for n, (a, b) in grads.items():
        if "pooler" in n or (rotary and "position_embeddings" in n):
            assert a is None
            continue
        assert (a.double() - b).norm() <= 2e-5 * b.norm() + 1e-7, n


def test_text_tower_refuses(ref):
    from ct_clip_amd import bert as product
    ids = torch.zeros(1, 40, dtype=torch.long)
    with pytest.raises(ValueError, match="position table"):
        product.bert_last_hidden_state(O.small_bert(), ids, None, torch.float32)
    with pytest.raises(NotImplementedError):
        product.bert_last_hidden_state(O.small_bert(position_embedding_type="relative_key"), ids[:, :8], None, torch.float32)
    with pytest.raises(ValueError):
        product.bert_last_hidden_state(O.small_bert(position_embedding_type="rotary", rotary_dim=33), ids, None, torch.float32)
