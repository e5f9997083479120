"""Rotary positions and windowed attention where a call can go wrong, without a device: the built code's waits, sizes of workspaces and grids, what a plan holds, options of the
text tower."""
import copy
import os
import re
import subprocess

import pytest
import torch

from ct_clip_amd import build
from ct_clip_amd import functional as Fn
from ct_clip_amd.bert import bert_last_hidden_state
from tests import long_report_oracle as O
from tests.test_long_reports_cpu import ref  # noqa: F401

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def windowed_kernels(tmp_path_factory):
    """{symbol: instructions (and None where a block begins)} of the built library's windowed attention kernels."""
    if not os.path.exists(OBJDUMP) or not os.path.exists(build.LIB):
        pytest.skip("needs the built library and llvm-objdump")
    where = tmp_path_factory.mktemp("isa")
    os.symlink(build.LIB, where / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=where, check=True, capture_output=True)
    kernels = {}
    for f in sorted(where.glob("*gfx950")):
        if b"3win" not in f.read_bytes():
            continue
        text = subprocess.run([OBJDUMP, "-d", "--symbolize-operands", str(f)], check=True, capture_output=True, text=True).stdout
        at = None
        for line in text.splitlines():
            m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
            if m and re.fullmatch(r"L\d+", m[1]):
                if at is not None:
                    at.append(None)
            elif m:
                at = kernels.setdefault(m[1], []) if "3win" in m[1] else None
            elif at is not None and line.startswith("\t"):
                at.append(line.split("//")[0].strip())
    return kernels


def test_a_tile_is_refilled_behind_the_reads_of_it(windowed_kernels):
    """Loads into LDS are not ordered with a wave's LDS reads: in the block that starts a refill, a wait for them stands in front."""
    seen = set()
    for name, code in windowed_kernels.items():
        for i, ins in enumerate(code):
            if not (ins and ins.startswith("buffer_load") and ins.endswith("lds")):
                continue
            seen.add(re.search(r"(fwd_kernel|rows_kernel|dq_kernel|dkv_kernel)", name)[1])
            back = i - 1
            while code[back] and not code[back].startswith(("ds_read", "s_branch", "s_cbranch")) and "lgkmcnt(0)" not in code[back]:
                back -= 1
            assert code[back] and "lgkmcnt(0)" in code[back], f"{name}: {code[back]} ... {ins}"
    assert seen == {"fwd_kernel", "rows_kernel", "dq_kernel", "dkv_kernel"}


# ------------------------------------------------------------------------------------------------------------- options of the text tower

YARN = dict(type="yarn", factor=8.0, original_length=512)
CONFIGS = [  # what BertConfig is given, what RotaryPositions of a head of 32 columns must be
    (dict(), dict()),
    (dict(rope_theta=500.0), dict(base=500.0)),
    (dict(rope_scaling=dict(type="linear", factor=4.0)), dict(scaling=dict(type="linear", factor=4.0))),
    (dict(rope_scaling=dict(rope_type="linear", factor=4.0), rope_theta=500.0, rotary_layout="interleaved"), dict(scaling=dict(type="linear", factor=4.0), base=500.0, layout="interleaved")),
    (dict(rope_scaling=dict(type="ntk", factor=4.0), rotary_dim=16), dict(scaling=dict(type="ntk", factor=4.0), dim=16)),
    (dict(rope_scaling=dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=512)), dict(scaling=YARN)),
    (dict(rope_scaling=dict(type="yarn", factor=8.0, original_length=256), rope_theta=500.0), dict(scaling=dict(YARN, original_length=256), base=500.0)),
    (dict(rope_scaling=dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=512, beta_fast=16.0, attention_factor=1.5, truncate=True)),
     dict(scaling=dict(YARN, beta_fast=16.0, attention_factor=1.5))),
    (dict(rope_parameters=dict(rope_type="default", rope_theta=500.0)), dict(base=500.0)),
    (dict(rope_parameters=dict(rope_type="linear", rope_theta=500.0, factor=2.0, partial_rotary_factor=0.5)), dict(scaling=dict(type="linear", factor=2.0), base=500.0, dim=16)),
]


def long_bert(**options):
    from transformers import BertConfig, BertModel
    torch.manual_seed(1)
    return BertModel(BertConfig(vocab_size=97, hidden_size=64, num_hidden_layers=1, num_attention_heads=2, intermediate_size=64, hidden_dropout_prob=0.0,
                                attention_probs_dropout_prob=0.0, position_embedding_type="rotary", **options))


@pytest.mark.parametrize("stored", ["constructed", "dict", "saved"])
@pytest.mark.parametrize("given,want", CONFIGS)
def test_options_as_the_config_s_constructor_keeps_them(ref, given, want, stored, tmp_path):
    """... and after a round trip through a dict or a file: the tower's output is that of the 64-bit form with the plan's frequencies."""
    from transformers import BertConfig
    model = long_bert(attention_window=(9, 4), attention_sinks=2, **given)
    if stored == "dict":
        model.config = BertConfig.from_dict(model.config.to_dict())
    elif stored == "saved":
        model.config.save_pretrained(tmp_path)
        model.config = BertConfig.from_pretrained(tmp_path)
    kw = dict(want)
    rope = Fn.RotaryPositions(kw.pop("dim", 32), **kw)
    ids = torch.randint(0, 97, (2, 50), generator=torch.Generator().manual_seed(2))
    got = bert_last_hidden_state(model, ids, None, torch.float32)
    plan = (torch.from_numpy(rope.frequencies), rope.magnitude, rope.dim, rope.interleaved)
    exact = O.bert64(copy.deepcopy(model).double(), ids, torch.ones_like(ids), plan, (9, 4), 2)
    torch.testing.assert_close(got.double(), exact, rtol=1e-5, atol=1e-5)          # one layer in f32: some 15 roundings of values of order 1


@pytest.mark.parametrize("scaling", [dict(rope_type="dynamic", factor=2.0), dict(rope_type="longrope", factor=2.0), dict(type="linear", rope_type="ntk", factor=2.0),
                                     dict(type="linear", factor=2.0, mscale=1.0), dict(rope_type="yarn", factor=2.0), dict(rope_type="default", mscale=1.0),
                                     dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=512, truncate=False), dict(rope_type="linear", factor=2.0, rope_theta=7.0)])
def test_options_that_the_tower_does_not_have_are_refused(ref, scaling):
    model = long_bert(rope_theta=500.0)
    model.config.rope_scaling = scaling
    with pytest.raises(ValueError):
        bert_last_hidden_state(model, torch.zeros((1, 4), dtype=torch.long), None, torch.float32)


# ------------------------------------------------------------------------------------------------------------------ the operators' calls

def test_a_dual_tensor_is_refused(ref):
    """Forward-mode derivatives: an error whether or not an input requires a gradient, never an output without a tangent; plain tensors pass at a dual level."""
    import torch.autograd.forward_ad as fwAD
    rope, x, m = Fn.RotaryPositions(32), torch.randn(6, 64), torch.zeros(6)
    calls = [lambda a, b: Fn.rotary(a, None, rope, 32), lambda a, b: Fn.rotary(b, a, rope, 32), lambda a, b: Fn.window_attention(a, b, b, 2, 32, window=2),
             lambda a, b: Fn.window_attention(b, a, b, 2, 32, window=2), lambda a, b: Fn.window_attention(b, b, a, 2, 32, window=2),
             lambda a, b: Fn.window_attention(a[:0], b, b, 2, 32, window=2)]
    for grad in (False, True):
        other = x.clone().requires_grad_(grad)
        for call in calls:
            want = call(x, other)
            with fwAD.dual_level():
                dual = fwAD.make_dual(x, torch.ones_like(x))
                with pytest.raises(NotImplementedError):
                    call(dual, other)
                with torch.no_grad(), pytest.raises(NotImplementedError):
                    call(dual, other)
                for a, b in zip(*(t if isinstance(t, tuple) else (t,) for t in (call(x, other), want))):
                    assert torch.equal(a, b)
        with fwAD.dual_level(), pytest.raises(NotImplementedError):
            Fn.window_attention(x, x, other, 2, 32, keymask=fwAD.make_dual(m, torch.ones_like(m)))


def test_workspace_of_one_long_sequence_among_many_short_ones():
    """Sequences without a row beyond their window take no room for the sinks: the partial sums are bounded by what the rows can hold, not by sequences times sinks."""
    from ct_clip_amd import _lib
    lib, H, D, left = _lib.load(), 12, 64, 256
    lengths = [8192] + [30] * 999
    seqs = Fn.PackedSequences(lengths)
    Mk = seqs.end

    def need(nseq, longest, M, sinks, ntiles):
        return lib.ctclip_win_attn_bwd_workspace(nseq, longest, longest, M, H, H, D, left, left, sinks, 0, ntiles)
    for sinks in (1, 4, 32, 512):
        s32 = (sinks + 31) // 32 * 32
        rows = Mk * s32 // (s32 + left - 30)
        one = 2 * rows * H * D * 4                      # a part of dK and dV in f32
        got = need(len(lengths), 8192, Mk, sinks, seqs.ntiles)
        assert one < got <= 2 * one, sinks              # the window's part and that of one chunk of rows
    # few sequences, or all of them long: as many rows as they have sinks
    assert need(12, 3001, 9688, 2, 84) == need(12, 3001, 9688, 2, 90)
    assert need(4, 2000, 8000, 4, 64) <= 2 * (1 + 11) * 4 * 32 * H * D * 4


def test_packed_sinks_partial_rows_do_not_meet():
    """The rule by which sequences take their rows: floor(first row * s32 / step), for any window, number of sinks and lengths."""
    import random
    rng = random.Random(5)
    for _ in range(300):
        left, sinks = rng.choice((0, 1, 7, 29, 30, 31, 64, 300)), rng.choice((1, 31, 32, 33, 100, 700))
        lengths = [rng.choice((0, 1, left, left + 1, left + 2, left + 3, left + 33, left + 34, left + 35, left + 66, rng.randint(1, 3000))) for _ in range(rng.randint(1, 60))]

        def keys(n):
            k = min(sinks, n - 1 - left)
            return (k + 31) // 32 * 32 if k > 0 else 0
        s32, M, first = max(map(keys, lengths)), sum(lengths), 0
        if not s32:
            continue
        step, end = min(s32 + left - 30, s32 // 32 * (left + 2)), 0
        for n in lengths:
            if keys(n):
                at = first * s32 // step
                assert at >= end
                end = at + keys(n)
            first += n
        assert end <= M * s32 // step


@pytest.mark.parametrize("cls_only", [False, True])
def test_statistics_are_kept_only_where_a_backward_pass_can_follow(ref, monkeypatch, cls_only):
    from tests.test_long_reports_cpu import RefOps
    asked, run = [], RefOps.win_attn_fwd
    monkeypatch.setattr(RefOps, "win_attn_fwd", lambda self, *a, want_lse=True, **kw: asked.append(want_lse) or run(self, *a, want_lse=want_lse, **kw))
    model, ids = long_bert(attention_window=3), torch.arange(16).view(2, 8)

    def tower():
        del asked[:]
        return bert_last_hidden_state(model, ids, None, torch.float32, cls_only=cls_only)
    out = tower()
    assert asked == [True] and out.requires_grad
    with torch.no_grad():
        assert torch.equal(tower(), out) and asked == [False]
    with torch.inference_mode():
        assert torch.equal(tower(), out) and asked == [False]
    model.requires_grad_(False)
    assert torch.equal(tower(), out) and asked == [False]
    model.requires_grad_(True)
    tower().square().sum().backward()
    assert all(p.grad is not None for n, p in model.named_parameters() if "pooler" not in n and "position" not in n)


def test_c_entries_refuse_a_grid_that_no_launch_holds():
    """2^32 threads along the first axis: every launch of a call is refused before the first one writes."""
    import ctypes
    from ct_clip_amd import _lib
    lib = _lib.load()
    buf = (ctypes.c_char * 512)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def fwd(nseq, L, H, D, dt=1, off=None, nt=0):
        M = nseq * L
        return lib.ctclip_win_attn_fwd(p, p, p, None, off, off, nt, p, None, None, nseq, L, L, M, M, H, H, D, 4, 4, 0, 0, H * D, H * D, H * D, H * D, 1.0, 0.0, 0, dt, None, 0, None)

    def bwd(nseq, L, H, Hk, D, dt=1, off=None, nt=0, sinks=0, ws=0):
        M = nseq * L
        return lib.ctclip_win_attn_bwd(p, p, p, None, off, off, nt, p, None, p, p, p, p, p, p, nseq, L, L, M, M, H, Hk, D, 4, 4, sinks, 0, H * D, Hk * D, Hk * D, H * D, H * D, H * D, Hk * D,
                                       Hk * D, 1.0, 0.0, 0, dt, p, ws, None)
    assert fwd(2 ** 21, 1, 8, 64) == -2 and b"2^32 threads" in lib.ctclip_last_error()           # few rows: a workgroup for a sequence and key head
    assert fwd(2 ** 20, 33, 16, 64, dt=0) == fwd(2 ** 21, 1, 8, 64, off=p, nt=2 ** 21) == -2     # tiles of rows
    assert bwd(2 ** 20, 3, 16, 2, 64) == bwd(2 ** 21, 1, 8, 1, 64, off=p, nt=2 ** 21) == -2      # dQ
    assert bwd(2 ** 20, 3, 8, 8, 128) == -2 and b"2^32 threads" in lib.ctclip_last_error()       # dK / dV, 512 threads
    assert bwd(2 ** 18, 40, 32, 32, 64, sinks=40, ws=2 ** 60) == -2                              # 2^23 workgroups of keys, and 2^24 of two sink blocks in front


def test_accumulators_of_split_passes_start_at_16_bytes():
    """They are written and read 16 bytes at a time; an odd number of rows stands in front of them twice."""
    from ct_clip_amd import _lib
    lib, odd = _lib.load(), 0
    for Lk in (768, 800, 2400, 5000, 32 * 37):
        for H, Lq, D in ((1, 1, 64), (3, 1, 32), (1, 33, 64), (5, 7, 128)):
            n = lib.ctclip_win_attn_fwd_workspace(1, Lq, Lk, H, H, D, -1, -1, 0, 0, 0) // 4
            rows = n // (D + 2)
            odd += rows % 2 and n > 0
            assert n % 4 == 0 and (n == 0 or n - rows * D >= 2 * rows)
    assert odd


@pytest.mark.parametrize("device", [torch.device("cuda", 0), torch.device("cuda"), "cuda"])
def test_tables_of_a_plan_are_recorded_on_the_streams_that_read_them(monkeypatch, device):
    """... and made before a capture, never inside one."""
    class Table:
        device = torch.device("cuda", 0)

        def __init__(self):
            self.read_on = []

        def to(self, device):
            return self

        def get_device(self):
            return 0

        def record_stream(self, stream):
            self.read_on.append(stream)
    now = dict(stream=7, capturing=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: now["stream"], raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: f"stream {now['stream']}")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now["capturing"])
    rope, seqs = Fn.RotaryPositions(32), Fn.PackedSequences([3, 200])
    rope._turns.host, seqs._tables.host = (Table(),), (Table(), Table())
    now["capturing"] = True
    for first in (rope.turns, seqs.on):
        with pytest.raises(RuntimeError, match="before the capture"):
            first(device)
    now["capturing"] = False
    tables = [rope.turns(device), *seqs.on(device)]
    rope.turns(device)
    assert [t.read_on for t in tables] == [[], [], []]
    now["stream"] = 9
    assert [rope.turns(device), *seqs.on(device)] == tables
    assert [t.read_on for t in tables] == [["stream 9"]] * 3
    now["capturing"] = True
    rope.turns(device)
    assert tables[0].read_on == ["stream 9"] * 2


def test_raw_strings_are_cut_at_the_model_s_text_length():
    import ct_clip_amd
    asked = []

    class Batch(dict):
        def to(self, device):
            return self

    def tokenizer(prompt, **kw):
        asked.append(kw)
        return Batch()

    def clip(**kw):
        return ct_clip_amd.CTCLIP(image_encoder=torch.nn.Identity(), text_encoder=long_bert(attention_window=3), dim_text=64, dim_image=32, dim_latent=32, tokenizer=tokenizer, **kw)
    for kw, n in ((dict(), 512), (dict(max_text_len=4096), 4096)):
        clip(**kw).tokenize("a report")
        assert asked.pop() == dict(return_tensors="pt", padding="max_length", truncation=True, max_length=n)


def test_reach_of_the_cls_row(ref):
    """Two layers of a window of 3 to the right: the [CLS] row depends on tokens 1 ... 6 and on none behind them."""
    from transformers import BertConfig, BertModel
    torch.manual_seed(3)
    model = BertModel(BertConfig(vocab_size=97, hidden_size=64, num_hidden_layers=2, num_attention_heads=2, intermediate_size=64, hidden_dropout_prob=0.0,
                                 attention_probs_dropout_prob=0.0, position_embedding_type="rotary", attention_window=(5, 3), initializer_range=0.3))
    ids = torch.arange(1, 13)[None]

    def cls(ids):
        with torch.no_grad():
            return bert_last_hidden_state(model, ids, None, torch.float32, cls_only=True)
    base = cls(ids)
    for j in range(1, 12):
        other = ids.clone()
        other[0, j] = 90
        assert torch.equal(cls(other), base) == (j > 6), j


@pytest.mark.parametrize("options", [dict(), dict(position_embedding_type="rotary", attention_window=3)])
def test_an_attention_mask_of_another_shape_is_refused(ref, options):
    """The kernels read one value for every token."""
    model, ids = O.small_bert(**options), torch.zeros((2, 9), dtype=torch.long)
    bert_last_hidden_state(model, ids, torch.ones(2, 9), torch.float32)
    for shape in ((2, 8), (1, 9), (9,), (2, 9, 1), (2, 10)):
        with pytest.raises(ValueError, match="attention_mask"):
            bert_last_hidden_state(model, ids, torch.ones(shape), torch.float32)


def test_lengths_that_the_c_entry_cannot_take_are_refused(ref):
    x, rope = torch.zeros(6, 64), Fn.RotaryPositions(32)
    for L in (2 ** 62, 2 ** 64 + 5):            # (the second one would arrive as 5)
        with pytest.raises(ValueError):
            Fn.rotary(x, None, rope, 32, L=L)
    Fn.rotary(x, None, rope, 32, L=2 ** 40)


def test_gradients_of_no_rows_reach_the_backend_row_by_row(ref, monkeypatch):
    """A sum's gradient is one number with strides of 0, which contiguous() keeps where there are no rows."""
    from tests.test_long_reports_cpu import RefOps
    strides = []
    monkeypatch.setattr(RefOps, "rotary", lambda self, q, k, *a, **kw: strides.append((q.stride(1), k.stride(1))) or (torch.zeros(q.shape), torch.zeros(k.shape)))
    x = torch.zeros((0, 64), requires_grad=True)
    q, k = Fn.rotary(x, x.detach().expand(0, 64), Fn.RotaryPositions(32), 32)
    torch.autograd.grad(q.sum() + k.sum(), x)
    y = torch.zeros((5, 64), requires_grad=True)
    q, k = Fn.rotary(y, y[:1, :1].expand(5, 64), Fn.RotaryPositions(32), 32)
    torch.autograd.grad(q.sum() + k.sum(), y)
    assert strides == [(1, 1)] * 4
