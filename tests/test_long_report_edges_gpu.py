"""Rotary positions and windowed attention on the device where a call can go wrong: one long sequence among many short ones, modes of autograd."""
import pytest
import torch

from ct_clip_amd import functional as Fn
from tests.test_long_reports_gpu import rnd, run_case

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths,first,H,Hk,D,window,sinks", [
    ([3] * 40 + [700] + [9] * 50 + [400, 1, 23, 0, 22], 0, 2, 1, 64, (20, 10), 40),       # a step of the smallest sequences: two blocks in 44 rows
    ([30] * 60 + [900] + [30] * 30, 5, 2, 2, 32, (100, 0), 4),                            # one block
    ([64] * 70 + [500, 66, 65, 98], 0, 4, 2, 128, (63, 20), 90),                          # just too short, and just long enough
    ([5] * 20 + [1500], 0, 1, 1, 64, (600, -1), 3),                                       # ... with the rows of a key tile split over workgroups
])
def test_sinks_of_packed_sequences_most_of_which_are_short(lengths, first, H, Hk, D, window, sinks, dtype):
    run_case(dtype, None, None, None, H, Hk, D, window, sinks, lengths=lengths, first=first, tail=2, seed=len(lengths))


@pytest.mark.parametrize("nseq,Lq,Lk,H,D,window,sinks,mask", [(8, 512, 512, 12, 64, (16, 16), 1, False), (8, 1, 512, 12, 64, (128, 128), 1, True), (2, 40, 40, 4, 32, (-1, -1), 0, False),
                                                              (4, 300, 300, 2, 128, (20, 3), 2, True), (2, 900, 900, 4, 64, (100, 100), 3, True), (1, 1, 9000, 8, 64, (-1, 0), 0, False)])
def test_the_output_s_bits_do_not_depend_on_the_mode(nseq, Lq, Lk, H, D, window, sinks, mask):
    """Forward for training, with frozen inputs and under no_grad: the same numbers."""
    q, k, v = rnd((nseq * Lq, H * D), BF16, 1), rnd((nseq * Lk, H * D), BF16, 2), rnd((nseq * Lk, H * D), BF16, 3)
    keymask = torch.where(torch.arange(nseq * Lk, device="cuda") % 7 == 3, torch.finfo(F32).min, 0.0) if mask else None

    def call():
        return Fn.window_attention(q, k, v, H, D, nseq=nseq, window=window, sinks=sinks, keymask=keymask, q_start=Lk - Lq)
    frozen = call()
    q.requires_grad_(True)
    trained = call()
    with torch.no_grad():
        assert torch.equal(call(), trained.detach())
    assert trained.requires_grad and torch.equal(frozen, trained.detach())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Lq,Lk,H,Hk,D", [(1, 768, 1, 1, 64), (1, 800, 3, 1, 32), (33, 768, 1, 1, 64), (7, 1184, 5, 5, 128)])
def test_split_passes_of_an_odd_number_of_rows(Lq, Lk, H, Hk, D, dtype):
    run_case(dtype, 1, Lq, Lk, H, Hk, D, (-1, -1), 0, q_start=Lk - Lq, seed=Lk)


def test_calls_from_several_threads():
    """First calls of kernels that need more than 64 KB of LDS, forward and backward, from eight threads at once, a stream each."""
    import threading
    q, k, v, do = (rnd((300, 2 * 128), F32, 3 + i) for i in range(4))
    out, start = [None] * 8, threading.Barrier(8)
    torch.cuda.synchronize()

    def call():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = Fn.window_attention(*leaves, 2, 128, window=50, sinks=2, dropout=(0.1, 9))
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            out[i] = call()
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    want = call()
    for got in out:
        assert got is not None and all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_plan_dropped_while_another_stream_still_reads_it():
    """What is allocated next on the stream that the plan was made on must not get the memory of its tables."""
    from ct_clip_amd import _lib
    x, lengths = rnd((700, 256), BF16, 1), [300, 1, 399]
    torch.cuda.synchronize()

    def calls(rope, seqs):
        return Fn.rotary(x, None, rope, 64, start=11), Fn.window_attention(x, x, x, 4, 64, nseq=seqs, window=9, sinks=2)
    want = calls(Fn.RotaryPositions(64), Fn.PackedSequences(lengths))
    side = torch.cuda.Stream()
    for _ in range(3):
        rope, seqs = Fn.RotaryPositions(64), Fn.PackedSequences(lengths)
        rope.turns(x.device), seqs.on(x.device)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            _lib.check(_lib.load().ctclip_spin(20000, side.cuda_stream), "ctclip_spin")          # 20 ms, under which the host runs ahead
            got = calls(rope, seqs)
        del rope, seqs
        import gc
        gc.collect()                     # (a plan of sequences and the geometries kept with it refer to each other)
        junk = [torch.full((n,), -1, dtype=torch.int32, device="cuda") for n in (64, 4, 14) * 20]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del junk


def test_tables_are_not_made_inside_a_capture():
    x = rnd((40, 64), BF16, 1)
    rope, seqs = Fn.RotaryPositions(64), Fn.PackedSequences([40])
    Fn.rotary(x, None, Fn.RotaryPositions(64), 64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x + 1
        with pytest.raises(RuntimeError, match="before the capture"):
            Fn.rotary(x, None, rope, 64)
        with pytest.raises(RuntimeError, match="before the capture"):
            Fn.window_attention(x, x, x, 1, 64, nseq=seqs)
    graph.replay()
    assert torch.equal(y, x + 1)
    assert torch.isfinite(Fn.rotary(x, None, rope, 64)).all()


def test_cls_rows_with_attention_dropout():
    """A tower in training mode: the last layer's [CLS] rows attended from alone draw the masks that they draw among all rows, forward and backward."""
    from transformers import BertConfig, BertModel
    from ct_clip_amd.bert import bert_last_hidden_state
    torch.manual_seed(0)
    bert = BertModel(BertConfig(vocab_size=50, hidden_size=128, num_hidden_layers=2, num_attention_heads=2, intermediate_size=128, position_embedding_type="rotary", attention_window=(20, 9),
                                attention_sinks=2, hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.3), add_pooling_layer=False).to("cuda").train()
    ids = torch.randint(0, 50, (3, 70), device="cuda")
    mask = (torch.arange(70, device="cuda")[None, :] < torch.tensor([[70], [41], [5]], device="cuda")).long()
    do = rnd((3, 128), F32, 4)
    runs = []
    for cls_only in (False, True, True):
        torch.manual_seed(5 if len(runs) < 2 else 6)
        x = bert_last_hidden_state(bert, ids, mask, F32, cls_only=cls_only)
        x = x if cls_only else x.view(3, 70, 128)[:, 0]
        names = [n for n, p in bert.named_parameters() if "position" not in n]
        grads = torch.autograd.grad(x, [p for n, p in bert.named_parameters() if "position" not in n], do)
        runs.append((x.detach(), dict(zip(names, grads))))
    tol = 2.0 ** -14                                                         # sums of up to 210 terms in another order (210 * 2^-24 < 2^-16), through two layers
    (a, ga), (b, gb), (c, _) = runs
    assert (a - b).abs().max() <= tol * a.abs().max()
    assert (b - c).abs().max() > 16 * tol * a.abs().max()                    # another seed, other masks: the comparison above would notice
    for n in ga:
        if "key.bias" not in n:                                              # (its true gradient is zero)
            assert (ga[n] - gb[n]).norm() <= 4 * tol * ga[n].norm() + 1e-6, n


@pytest.mark.parametrize("options", [dict(attention_window=6), dict(attention_window=(3, -1), attention_sinks=2, rope_scaling=dict(type="linear", factor=2.0), rotary_layout="interleaved")])
def test_training_step_of_a_tower_of_long_reports_replayed(golden, tmp_path, options):
    """The trainer's step captured into a graph with the tower's options on: replays continue three eager steps bit for bit, with dropout they draw fresh masks."""
    import ct_clip_amd
    from ct_clip_amd.trainer import GraphedStep
    from tests.helpers import TextBatch, build_model
    g = golden("tiny")
    text, video = TextBatch(g["input_ids"].to("cuda"), g["attention_mask"].to("cuda")), g["video"].to("cuda")

    def run(n_eager, n_graph, dropout):
        clip = build_model(g["config"], g["state_dict"], "cuda", BF16)
        cfg = clip.text_transformer.config
        for name, value in dict(options, position_embedding_type="rotary", hidden_dropout_prob=dropout, attention_probs_dropout_prob=dropout).items():
            setattr(cfg, name, value)
        clip.train()
        tr = ct_clip_amd.CTClipTrainer(clip, num_train_steps=10, batch_size=2, tokenizer=object(), lr=1e-3, train_dataset=[0], evaluate=False, checkpoint=False,
                                       results_folder=str(tmp_path / f"res{n_graph}{dropout}"), num_workers=0)
        table = clip.text_transformer.embeddings.position_embeddings.weight.detach().clone()
        torch.manual_seed(11)
        losses = []
        for _ in range(n_eager):
            losses.append(tr.forward_backward(video, text).detach().clone())
            tr.optim.step(tr.max_grad_norm)
            tr.optim.zero_grad()
        if n_graph:
            gs = GraphedStep(tr).capture(video, text)
            try:
                for _ in range(n_graph):
                    losses.append(gs.run().detach().clone())
            finally:
                gs.close()
        torch.cuda.synchronize()
        assert torch.equal(table, clip.text_transformer.embeddings.position_embeddings.weight)
        return torch.stack(losses).flatten().tolist(), tr.optim.flat_param.clone(), tr.optim.exp_avg.clone()
    la, pa, ma = run(6, 0, 0.0)
    lb, pb, mb = run(3, 3, 0.0)
    assert la == lb and torch.equal(pa, pb) and torch.equal(ma, mb) and torch.isfinite(pa).all()
    assert len(set(run(3, 3, 0.1)[0][3:])) == 3


def test_tables_on_a_device_named_without_an_index():
    """Made ahead of a capture by whoever holds the plan."""
    x, rope, seqs = rnd((40, 64), BF16, 1), Fn.RotaryPositions(64), Fn.PackedSequences([40])
    for device in ("cuda", torch.device("cuda"), x.device):
        for _ in range(2):
            assert rope.turns(device).device == x.device and seqs.on(device)[0].device == x.device
    assert torch.isfinite(Fn.rotary(x, None, rope, 64)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forms_of_arguments(dtype):
    """Key masks of other types and shapes, misaligned and expanded tensors, a gradient that is one number expanded, dropout of probability 0: the same as their plain forms."""
    n, L, H, D = 2, 70, 2, 32
    q, k, v = (rnd((n * L, H * D), dtype, i) for i in (1, 2, 3))
    mask = torch.zeros((n, L), device="cuda")
    mask[0, 40:] = torch.finfo(F32).min
    mask[1, ::3] = -2.5

    def call(q=q, k=k, v=v, keymask=mask, **kw):
        return Fn.window_attention(q, k, v, H, D, nseq=n, window=(9, 5), sinks=2, keymask=keymask, **kw)
    want = call()
    for m in (mask.double(), mask.bfloat16(), mask[:, None, None, :], mask.reshape(-1), mask.t().contiguous().t(), mask.clone().requires_grad_(True)):
        assert torch.equal(call(keymask=m), want)
    assert torch.equal(call(dropout=(0.0, 3)), want)

    def odd(t):          # one element off a 16-byte row
        wide = torch.zeros((t.shape[0], t.shape[1] + 3), dtype=t.dtype, device="cuda")
        wide[:, 1:-2] = t
        return wide[:, 1:-2]
    assert torch.equal(call(odd(q), odd(k), odd(v)), want)
    one = [t[:1].clone().requires_grad_(True) for t in (k, v)]
    full = [t.detach().expand(n * L, -1).contiguous().requires_grad_(True) for t in one]
    a, b = call(k=one[0].expand(n * L, -1), v=one[1].expand(n * L, -1)), call(k=full[0], v=full[1])
    assert torch.equal(a, b)
    ga, gb = torch.autograd.grad(a.sum(), one), torch.autograd.grad(b, full, torch.ones_like(b))
    assert all(torch.equal(x, y.sum(0, keepdim=True)) for x, y in zip(ga, gb))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_calls_without_rows(dtype):
    rope, none, keys = Fn.RotaryPositions(32), torch.zeros((0, 64), dtype=dtype, device="cuda", requires_grad=True), rnd((12, 64), dtype, 1).requires_grad_(True)
    q, k = Fn.rotary(none, none, rope, 32, L=4, start=9)
    assert q.shape == k.shape == (0, 64)
    (g,) = torch.autograd.grad(q.sum() + k.sum(), none)
    assert g.shape == (0, 64)
    o = Fn.window_attention(none, keys, keys, 2, 32, nseq=3, window=2)
    g0, g1 = torch.autograd.grad(o.sum(), (none, keys))
    assert o.shape == g0.shape == (0, 64) and not g1.any()
    assert Fn.window_attention(none, none, none, 2, 32, nseq=0).shape == (0, 64)
    assert Fn.window_attention(none, none, none, 2, 32, nseq=Fn.PackedSequences([])).shape == (0, 64)
    o = Fn.window_attention(keys, keys, keys, 2, 32, nseq=Fn.PackedSequences([0, 0], first=3))
    (g,) = torch.autograd.grad(o.sum(), keys)
    assert not o.any() and not g.any()


def test_packed_training_captured_and_replayed_and_a_second_backward_pass():
    """Rows outside the sequences, sinks of one long sequence among short ones, a key mask: each replay equals the eager result; so does the same graph's second backward pass."""
    H, D, lengths = 2, 64, [30] * 20 + [700] + [1, 0, 45]
    seqs = Fn.PackedSequences(lengths, first=4)
    M = seqs.end + 9
    q, k, v, do = (rnd((M, H * D), BF16, i) for i in range(4))
    mask = torch.zeros(M, device="cuda")
    rope = Fn.RotaryPositions(32, layout="interleaved")
    positions = torch.cat([torch.zeros(4, dtype=torch.int64)] + [torch.arange(n) for n in lengths] + [torch.zeros(9, dtype=torch.int64)]).to("cuda")

    def step(again=False):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        a, b = Fn.rotary(leaves[0], leaves[1], rope, D, positions=positions)
        o = Fn.window_attention(a, b, leaves[2], H, D, nseq=seqs, window=(60, 20), sinks=3, keymask=mask)
        grads = torch.autograd.grad(o, leaves, do, retain_graph=again)
        if again:
            assert all(torch.equal(x, y) for x, y in zip(grads, torch.autograd.grad(o, leaves, do)))
        return [o.detach(), *grads]
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
        for i, t in enumerate((q, k, v, do)):
            t.copy_(rnd(tuple(t.shape), BF16, 80 + 4 * rep + i))
        mask[rep::5] = torch.finfo(F32).min
        want = step(again=True)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert not any(t[:4].any() or t[seqs.end:].any() for t in out)
