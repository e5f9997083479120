"""Text tower: forward/backward of a HuggingFace ``BertModel`` on the gfx950 kernels.

The reference calls ``self.text_transformer(input_ids, attention_mask=...)[0]`` (CT_CLIP/ct_clip/ct_clip.py:685-686) on a
``transformers.BertModel`` (scripts/run_train.py:9).  Here the HF module is kept as the *parameter container* (so
``state_dict`` keys ``text_transformer.*`` are unchanged) and its arithmetic -- embeddings gather, post-LN encoder layers
with biased dense projections, softmax attention with key-padding mask, erf-GELU FFN (HF modeling_bert.py: BertEmbeddings,
BertSelfAttention, BertSelfOutput, BertIntermediate, BertOutput) -- runs through ``ct_clip_amd.functional``.
The pooler is skipped: CT-CLIP discards it (ct_clip.py:686,762).

Reports longer than the position table (512 rows), all as attributes of the HF config (``BertConfig(..., position_embedding_type="rotary", attention_window=256)``):
  position_embedding_type = "rotary"   rotary positions on q and k instead of the absolute table (which is then neither read nor trained); rotary_dim (default: the whole
                                       head), rope_theta (10000), rotary_layout ("half" | "interleaved"), rope_scaling (dict; by HF's names, as transformers 5 keeps them in
                                       config.rope_parameters too: "rope_type" "default" | "linear" | "ntk" | "yarn", "factor", for yarn
                                       "original_max_position_embeddings", or by those of ``functional.RotaryPositions``);
  attention_window = n or (l, r)       every token attends within its window, cost linear in the length; attention_sinks first tokens (default 1: [CLS]) stay visible.
What reaches the latent: CT-CLIP reads the [CLS] row alone.  A sink is seen by every token but sees no more than they do: [CLS] itself sees the r tokens behind it, and through n
layers the first n * r; the words after those have no part in the latent.  Choose the window by the longest report.
"""
import math

import torch

from . import functional as Fn

def is_hf_bert(module):
    return hasattr(module, "embeddings") and hasattr(module, "encoder") and hasattr(module.encoder, "layer") \
        and hasattr(module.embeddings, "word_embeddings")


def _rope_options(cfg, dh):
    """-> (rotated columns, base, layout, scaling of ``functional.RotaryPositions`` or None) from the config, whose constructor rewrites the dict: transformers 5 adds "rope_type" to it,
    the base and, for yarn, the length of the original context, and reads and writes it as rope_parameters too."""
    given = {name: value for name, value in dict(getattr(cfg, "rope_scaling", None) or getattr(cfg, "rope_parameters", None) or {}).items() if value is not None}
    kinds = {given.pop(name) for name in ("rope_type", "type") if name in given}
    if len(kinds) > 1:
        raise ValueError(f"rope_scaling: two types, {sorted(kinds)}")
    kind = kinds.pop() if kinds else "default"
    bases = {float(b) for b in (given.pop("rope_theta", None), getattr(cfg, "rope_theta", None)) if b}
    if len(bases) > 1:
        raise ValueError(f"rope_theta: two values, {sorted(bases)}, beside rope_scaling and in it")
    part = given.pop("partial_rotary_factor", None)
    dim = getattr(cfg, "rotary_dim", None) or (int(dh * part) if part is not None else dh)
    if kind in ("default", "none"):
        given.pop("factor", None)
    if kind == "yarn":
        original = given.pop("original_max_position_embeddings", None)          # (transformers' own: the position table's rows unless the caller said so)
        given.setdefault("original_length", original)
        if given.pop("truncate", True) is not True:
            raise ValueError("rope_scaling yarn: truncate = False is not implemented")
    scaling = None if kind in ("default", "none") and not given else dict(given, type=kind)
    return dim, bases.pop() if bases else 10000.0, getattr(cfg, "rotary_layout", None) or "half", scaling


def _long_report_options(bert, dh):
    """-> (RotaryPositions or None, (left, right) or None, sinks) from the config."""
    cfg = bert.config
    kind = getattr(cfg, "position_embedding_type", "absolute") or "absolute"
    if kind not in ("absolute", "rotary"):
        raise NotImplementedError("only absolute and rotary position embeddings are implemented")
    rope = None
    if kind == "rotary":
        key = _rope_options(cfg, dh)
        held = bert.__dict__.get("_ctclip_rope")
        if held is None or held[0] != key:
            held = bert.__dict__["_ctclip_rope"] = (key, Fn.RotaryPositions(key[0], base=key[1], layout=key[2], scaling=key[3]))
        rope = held[1]
    window = getattr(cfg, "attention_window", None)
    if window is not None:
        window = (int(window), int(window)) if not isinstance(window, (tuple, list)) else (int(window[0]), int(window[1]))
    sinks = getattr(cfg, "attention_sinks", None)
    return rope, window, 1 if sinks is None else int(sinks)


def bert_last_hidden_state(bert, input_ids, attention_mask, dtype, operand_dtype=None, cls_only=False):
    """Returns last_hidden_state as a (B*T, hidden) activation in ``dtype`` -- or, with cls_only, its rows of the [CLS] positions, (B, hidden).

    cls_only: CT-CLIP reads enc_text[:, 0, :] and nothing else (ct_clip.py:762), so in the LAST layer only the [CLS] rows of the attention output
    have a consumer: the attention output projection, both LayerNorms, the feed-forward block, their dropouts and all their backward run on B rows
    instead of B*T (9 of the 12 d^2 multiply-adds per token of that layer; the q | k | v projection and the attention core still see every
    token: the keys and values of all positions feed the [CLS] query).  Same numbers for every consumer of the [CLS] rows, same parameter gradients.

    operand_dtype (mixed precision, the default of the bf16 mode: dtype = f32, operand_dtype = bf16): the residual stream, both
    LayerNorms of a layer, bias / dropout / residual adds, GELU and every GEMM's accumulate-and-store are f32 -- what torch.autocast
    keeps in f32 around an HF BertModel -- and bf16 appears only where the matrix cores read it: the GEMM operands (each f32 activation
    rounded once on its way into a GEMM), q | k | v and the attention core.  M = B*T rows x 768: the f32 tensors are a few MB."""
    od = operand_dtype if (operand_dtype is not None and operand_dtype != dtype) else None
    cfg = bert.config
    if getattr(cfg, "hidden_act", "gelu") != "gelu":
        raise NotImplementedError(f"hidden_act={cfg.hidden_act!r}: only erf-GELU BERT is implemented")
    rope, window, sinks = _long_report_options(bert, cfg.hidden_size // cfg.num_attention_heads)
    # train-mode dropout (HF modeling_bert.py: BertEmbeddings, BertSelfAttention, BertSelfOutput, BertOutput).  Masks are
    # counter-based (Philox, ct_clip_amd/csrc/common.h): one 62-bit seed per forward drawn from torch's CPU generator (so that
    # torch.manual_seed reproduces a run), call sites separated by stream ids / seed offsets, regenerated in backward.
    p_hid = float(cfg.hidden_dropout_prob) if bert.training else 0.0
    p_att = float(cfg.attention_probs_dropout_prob) if bert.training else 0.0
    seed = int(torch.randint(0, 2 ** 62, (1,)).item()) if (p_hid > 0 or p_att > 0) else 0

    def drop(h, residual, site):   # only reached with p_hid > 0, except for the embeddings (identity then)
        return Fn.DropoutAddFn.apply(h, residual, p_hid, seed, site) if p_hid > 0 else h
    emb = bert.embeddings
    dev = emb.word_embeddings.weight.device
    ids = input_ids.to(dev).contiguous()
    Bsz, T = ids.shape
    nh = cfg.num_attention_heads
    hidden = cfg.hidden_size
    dh = hidden // nh
    eps = cfg.layer_norm_eps

    if rope is None and T > emb.position_embeddings.weight.shape[0]:
        raise ValueError(f"{T} tokens, and {emb.position_embeddings.weight.shape[0]} rows in the position table (config.position_embedding_type = \"rotary\" has none)")
    x = Fn.BertEmbedFn.apply(ids, emb.word_embeddings.weight, emb.position_embeddings.weight if rope is None else None,
                             emb.token_type_embeddings.weight, dtype)
    x = Fn.layer_norm(x, emb.LayerNorm.weight, emb.LayerNorm.bias, eps)
    x = drop(x, None, 0)
    keymask = None
    if attention_mask is not None:
        if attention_mask.shape != ids.shape:
            raise ValueError(f"attention_mask {tuple(attention_mask.shape)} for input_ids {tuple(ids.shape)}")
        # additive key mask, as HF builds it: (1 - mask) * finfo.min
        keymask = ((1.0 - attention_mask.to(device=dev, dtype=torch.float32)) * torch.finfo(torch.float32).min).contiguous()
    scale = 1.0 / math.sqrt(dh)
    nlayers = len(bert.encoder.layer)
    for li, layer in enumerate(bert.encoder.layer):
        x = Fn.grad_ready(x, layer)
        sa, so = layer.attention.self, layer.attention.output
        # (x feeds the attention AND the residual connection: the node hands back a view of x for the latter, so that in backward the residual
        # path's gradient is added inside the grad-input GEMM's epilogue instead of by an elementwise accumulation kernel)
        drop_att = (p_att, seed + 1 + li) if p_att > 0 else None
        last_cls = cls_only and li == nlayers - 1 and T > 1
        qkv_args = (x, sa.query.weight, sa.key.weight, sa.value.weight, sa.query.bias, sa.key.bias, sa.value.bias, keymask, Bsz, T, nh, dh, scale, drop_att)
        if rope is None and window is None:
            c, x_res = Fn.QkvSdpaFn.apply(*qkv_args, od, True)
        else:
            c, x_res = Fn.QkvWindowFn.apply(*qkv_args, rope, window or (-1, -1), sinks if window else 0, last_cls, od, True, torch.is_grad_enabled())
        if last_cls:
            # rows b * T of the attention output and of the layer input: everything behind them in this layer is row-wise
            if c.shape[0] != Bsz:
                c = c.view(Bsz, T * c.shape[1])[:, :c.shape[1]].contiguous()
            x_res = x_res.view(Bsz, T * hidden)[:, :hidden].contiguous()
        if p_hid > 0:    # dense -> dropout -> + input -> LayerNorm
            h1 = drop(Fn.linear(c, so.dense.weight, so.dense.bias, out_dtype=dtype, operand_dtype=od), x_res, 1 + 2 * li)
        else:
            h1 = Fn.linear(c, so.dense.weight, so.dense.bias, residual=x_res, out_dtype=dtype, operand_dtype=od)
        x = Fn.layer_norm(h1, so.LayerNorm.weight, so.LayerNorm.bias, eps)
        u, x_res = Fn.linear(x, layer.intermediate.dense.weight, layer.intermediate.dense.bias, operand_dtype=od, passthrough=True)
        m = Fn.GeluFn.apply(u)
        if p_hid > 0:
            h2 = drop(Fn.linear(m, layer.output.dense.weight, layer.output.dense.bias, operand_dtype=od), x_res, 2 + 2 * li)
        else:
            h2 = Fn.linear(m, layer.output.dense.weight, layer.output.dense.bias, residual=x_res, operand_dtype=od)
        x = Fn.layer_norm(h2, layer.output.LayerNorm.weight, layer.output.LayerNorm.bias, eps)
    return x
