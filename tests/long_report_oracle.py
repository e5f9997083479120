"""Plain 64-bit forms of rotary positions and windowed attention, with elementwise error bounds (test infrastructure).

The bounds count roundings: `ut` is half a step of the tensors' type relative to a value (bf16 2^-8, f32 2^-24), `u` that of the f32 the kernels accumulate in.
A sum of n products in f32 is off by at most (n + 2) u times the sum of the products' magnitudes."""
import math

import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------------------------ rotary

def rotary64(x, freq, magnitude, D, rot, interleaved, pos, inverse=False):
    """-> (rotated x in 64 bits, sum of the magnitudes of the two products of every element)."""
    x = x.double().reshape(x.shape[0], -1, D)
    ang = pos.double()[:, None] * freq[None, :].to(x.device)
    c, s = torch.cos(ang)[:, None] * magnitude, torch.sin(ang)[:, None] * magnitude * (-1 if inverse else 1)
    ia = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    ib = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    a, b = x[..., ia], x[..., ib]
    y, m = x.clone(), torch.zeros_like(x)
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    m[..., ia] = m[..., ib] = (a.abs() + b.abs()) * magnitude
    return y.reshape(x.shape[0], -1), m.reshape(x.shape[0], -1)


def rotary_bound(y, m, dtype):
    """cos and sin: the angle within a quarter turn is rounded twice (0.8 * 2 u), its polynomials four times (4 u), the product with the magnitude once, the two products
    of an element and their sum three times: 10 u of |a| + |b| in all, 2^-33 turns of the angle itself, and the rounding of the result."""
    return m * (10 * U32 + 2.0 ** -33 * 2 * math.pi) + half_step(dtype) * y.abs()


# --------------------------------------------------------------------------------------------------------------- attention

def visible(Lq, Lk, left, right, sinks, q_start, device="cpu"):
    i = q_start + torch.arange(Lq, device=device)[:, None]
    j = torch.arange(Lk, device=device)[None, :]
    see = torch.ones((Lq, Lk), dtype=torch.bool, device=device)
    if right >= 0:
        see &= j <= i + right
    if left >= 0:
        see &= (j >= i - left) | (j < sinks)
    return see


def attention64(q, k, v, H, Hk, D, see, mask, scale, dout=None, drop=None, dtype=torch.float32):
    """One sequence.  q (Lq, H D), k | v (Lk, Hk D); see (Lq, Lk); mask (Lk) additive or None; drop (H, Lq, Lk) multipliers or None.
    -> {"o": (value, bound), and with dout "dq", "dk", "dv"}; everything in 64 bits."""
    Lq, Lk, G, ut = q.shape[0], k.shape[0], H // Hk, half_step(dtype)
    if mask is not None:
        mask = mask.double()
        shown = mask > -1e30                                     # (NaN hides)
        see = see & shown[None, :]
        mask = torch.where(shown, mask, torch.zeros_like(mask))
        k, v = (torch.where(shown[:, None], t, torch.zeros_like(t)) for t in (k, v))
    Q = q.double().reshape(Lq, H, D).transpose(0, 1)
    K, V = (t.double().reshape(Lk, Hk, D).transpose(0, 1).repeat_interleave(G, 0) for t in (k, v))
    S = Q @ K.transpose(1, 2).contiguous() * scale
    top = (Q.abs() @ K.abs().transpose(1, 2).contiguous() * scale).masked_fill(~see, 0.0).amax(-1, keepdim=True) if Lk else S.new_zeros((H, Lq, 1))
    if mask is not None:
        S = S + mask[None, None, :]
        top = top + mask.abs().max() if Lk else top
    S = S.masked_fill(~see, -math.inf)
    empty = ~see.any(-1)
    P = torch.softmax(S.masked_fill(empty[None, :, None], 0.0), -1).masked_fill(~see, 0.0)
    Pd = P if drop is None else P * drop.double()
    n = Lk
    O, A = Pd @ V, Pd @ V.abs()
    # a probability: its score is off by (D + 4) u of the sum of |q k| (and the mask and the maximum by one rounding each), hence exp2 and the sum; rounded to the operand type
    ep = (ut + U32 * (2 * (D + 6) * top + n + 16))
    eo = 1.01 * (ep * A + ut * O.abs())

    def rows(x):
        return x.transpose(0, 1).reshape(x.shape[1], -1)

    def shared(x):
        return rows(x.reshape(Hk, G, Lk, D).sum(1))
    out = {"o": (rows(O), rows(eo))}
    if dout is None:
        return out
    dO = dout.double().reshape(Lq, H, D).transpose(0, 1)
    dP = dO @ V.transpose(1, 2).contiguous()
    aP = dO.abs() @ V.abs().transpose(1, 2).contiguous()
    delta = (dO * O).sum(-1, keepdim=True)
    if drop is not None:
        dP, aP = dP * drop.double(), aP * drop.double()
    dS = P * (dP - delta)
    # Delta is taken of the rounded output; dP is an f32 sum of D products
    edelta = (dO.abs() * eo).sum(-1, keepdim=True) + (D + 2) * U32 * (dO.abs() * O.abs()).sum(-1, keepdim=True)
    epf = U32 * (2 * (D + 6) * top + n + 16)
    edS = 1.01 * ((ut + epf + 2 * U32) * dS.abs() + P * ((D + 2) * U32 * aP + edelta) + U32 * P * (dP.abs() + delta.abs()))
    rowsum = (Lq * G + 8) * U32
    out["dq"] = tuple(map(rows, (dS @ K * scale, 1.01 * (scale * ((edS + (n + 4) * U32 * dS.abs()) @ K.abs()) + ut * (dS @ K * scale).abs()))))
    tS, tP, tE = dS.transpose(1, 2).contiguous(), Pd.transpose(1, 2).contiguous(), edS.transpose(1, 2).contiguous()
    dk, dv = shared(tS @ Q * scale), shared(tP @ dO)
    out["dk"] = (dk, 1.01 * (shared((tE + rowsum * tS.abs()) @ Q.abs() * scale) + ut * dk.abs()))
    eP = ((ep + rowsum) * Pd).transpose(1, 2).contiguous()
    out["dv"] = (dv, 1.01 * (shared(eP @ dO.abs()) + ut * dv.abs()))
    return out


def batch64(q, k, v, H, Hk, D, spans, left, right, sinks, q_start, keymask, scale, dout=None, drop=None, dtype=torch.float32):
    """Sequences given as (q0, Lq, k0, Lk) rows; keymask flat per key row.  Rows outside are 0 (bound 0)."""
    names = ("o",) if dout is None else ("o", "dq", "dk", "dv")
    like = {"o": q, "dq": q, "dk": k, "dv": v}
    res = {n: [torch.zeros(like[n].shape, dtype=torch.float64, device=q.device) for _ in range(2)] for n in names}
    for b, (q0, lq, k0, lk) in enumerate(spans):
        if lq == 0:
            continue
        r = attention64(q[q0:q0 + lq], k[k0:k0 + lk], v[k0:k0 + lk], H, Hk, D, visible(lq, lk, left, right, sinks, q_start, q.device),
                        keymask[k0:k0 + lk] if keymask is not None else None, scale, dout[q0:q0 + lq] if dout is not None else None,
                        drop[b][:, :lq, :lk] if drop is not None else None, dtype)
        for n in names:
            at = slice(q0, q0 + lq) if n in ("o", "dq") else slice(k0, k0 + lk)
            for t, x in zip(res[n], r[n]):
                t[at] = x
    return res


def check(got, want, what):
    """Every element within its bound (a quarter of the smallest f32 normal absolute: exact zeros have bound 0)."""
    value, bound = want
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - value).abs() - bound
    worst = over.max().item() if over.numel() else 0.0
    if worst > 2.0 ** -128:
        at = (over == over.max()).nonzero()[0].tolist()
        raise AssertionError(f"{what}: {at}: got {got[tuple(at)].item():.9g}, want {value[tuple(at)].item():.9g}, bound {bound[tuple(at)].item():.3g}, "
                             f"{(over > 2.0 ** -128).sum().item()} of {over.numel()} over")


# ------------------------------------------------------------------------------------------------------------- text tower

def bert64(model, ids, attention_mask, rope=None, window=None, sinks=0):
    """Last hidden state (B T, hidden) of a BertModel of doubles with rotary positions and / or windowed attention, differentiable, no dropout.
    rope = (frequencies, magnitude, rot, interleaved)."""
    import torch.nn.functional as F
    cfg, emb = model.config, model.embeddings
    B, T = ids.shape
    H, hid = cfg.num_attention_heads, cfg.hidden_size
    D = hid // H
    x = emb.word_embeddings.weight[ids] + emb.token_type_embeddings.weight[0]
    if rope is None:
        x = x + emb.position_embeddings.weight[:T]
    x = F.layer_norm(x, (hid,), emb.LayerNorm.weight, emb.LayerNorm.bias, cfg.layer_norm_eps).reshape(B * T, hid)
    left, right = window if window is not None else (-1, -1)
    see = visible(T, T, left, right, sinks, 0, x.device)[None, None] & (attention_mask.reshape(B, 1, 1, T) > 0)
    pos = torch.arange(B * T, device=x.device) % T
    for layer in model.encoder.layer:
        sa, so = layer.attention.self, layer.attention.output
        q, k, v = (m(x) for m in (sa.query, sa.key, sa.value))
        if rope is not None:
            q, k = (rotary64(t, rope[0], rope[1], D, rope[2], rope[3], pos)[0] for t in (q, k))
        q, k, v = (t.reshape(B, T, H, D).transpose(1, 2) for t in (q, k, v))
        s = (q @ k.transpose(-1, -2).contiguous() / math.sqrt(D)).masked_fill(~see, -1e300)
        p = torch.softmax(s, -1).masked_fill(~see, 0.0)
        c = (p @ v).transpose(1, 2).reshape(B * T, hid)
        x = F.layer_norm(so.dense(c) + x, (hid,), so.LayerNorm.weight, so.LayerNorm.bias, cfg.layer_norm_eps)
        m = F.gelu(layer.intermediate.dense(x))
        x = F.layer_norm(layer.output.dense(m) + x, (hid,), layer.output.LayerNorm.weight, layer.output.LayerNorm.bias, cfg.layer_norm_eps)
    return x


def small_bert(seed=0, heads=2, hidden=64, layers=2, **options):
    from transformers import BertConfig, BertModel
    torch.manual_seed(seed)
    model = BertModel(BertConfig(vocab_size=97, hidden_size=hidden, num_hidden_layers=layers, num_attention_heads=heads, intermediate_size=2 * hidden,
                                 max_position_embeddings=32, hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0))
    with torch.no_grad():
        for p in model.parameters():         # (the initial 0.02 makes every attention uniform)
            p.add_(torch.randn_like(p) * (0.3 / math.sqrt(p.shape[-1]) if p.ndim > 1 else 0.1))
    for name, value in options.items():
        setattr(model.config, name, value)
    return model


BERT_OPTIONS = [
    dict(position_embedding_type="rotary"),
    dict(position_embedding_type="rotary", rotary_dim=16, rotary_layout="interleaved", rope_theta=500.0, rope_scaling=dict(type="yarn", factor=4.0, original_length=32),
         attention_window=7),
    dict(position_embedding_type="rotary", attention_window=(20, 3), attention_sinks=4),
    dict(attention_window=5),
]


def bert_case(options, T, device, B=3, cls_only=False, dtype=torch.float32, operand_dtype=None):
    """-> (hidden, {name: gradient}) of the product and of the 64-bit form for the same weights and output gradient."""
    import copy
    from ct_clip_amd import bert as product
    from ct_clip_amd import functional as Fn
    model = small_bert(seed=T, **options)
    plain = copy.deepcopy(model).double().to(device)
    model = model.to(device)
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(0, 97, (B, T), generator=g).to(device)
    mask = (torch.arange(T)[None, :] < torch.tensor([T, max(1, T // 2), max(1, T - 3)])[:, None]).long().to(device)
    D = model.config.hidden_size // model.config.num_attention_heads
    rope = None
    if options.get("position_embedding_type") == "rotary":
        r = Fn.RotaryPositions(options.get("rotary_dim") or D, base=options.get("rope_theta", 10000.0), layout=options.get("rotary_layout", "half"), scaling=options.get("rope_scaling"))
        rope = (torch.from_numpy(r.frequencies), r.magnitude, r.dim, r.layout == "interleaved")
    window = options.get("attention_window")
    window = (window, window) if isinstance(window, int) else window
    want = bert64(plain, ids, mask, rope, window, options.get("attention_sinks", 1) if window is not None else 0)
    got = product.bert_last_hidden_state(model, ids, mask, dtype, operand_dtype, cls_only=cls_only)
    if cls_only:
        want = want.reshape(B, T, -1)[:, 0]
    do = torch.randn(tuple(want.shape), generator=g).to(device)
    (got * do.to(got.dtype)).sum().backward()
    (want * do.double()).sum().backward()
    other = dict(plain.named_parameters())
    grads = {n: (p.grad, other[n].grad) for n, p in model.named_parameters()}
    return got, want, grads, rope is not None
