"""Autograd nodes of the text tower's attention on a torch backend: values and gradients against the 64-bit form."""
import pytest
import torch

from ct_clip_amd import backend
from ct_clip_amd import functional as Fn
from tests import long_report_oracle as O
from tests.ref_backend import RefBackend

SDPA = [  # nseq, L, H, D, key mask, dropout
    (2, 77, 2, 64, True, None),
    (1, 64, 3, 64, False, None),
    (3, 33, 2, 32, True, (0.2, 5)),
    (2, 24, 1, 32, False, (0.1, 6)),
]


def sdpa_case(device, dtype, nseq, L, H, D, masked, dropout):
    """Checks the output and the gradients of ``SdpaFn``, every element within its bound."""
    g = torch.Generator().manual_seed(L)
    q, k, v, do = (torch.randn((nseq * L, H * D), generator=g).to(device).to(dtype) for _ in range(4))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    mask = None
    if masked:
        shown = torch.arange(L)[None, :] < torch.tensor([L, L - L // 3, L // 2])[:nseq, None]
        mask = ((1.0 - shown.float()) * torch.finfo(torch.float32).min).to(device)
    o = Fn.SdpaFn.apply(*leaves, mask, nseq, L, H, D, D ** -0.5, dropout)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, do)), o=o.detach())
    drop = backend.get().attn_dropout_mask(nseq, H, L, *dropout, torch.device(device)) if dropout else None
    want = O.batch64(q.detach(), k.detach(), v.detach(), H, H, D, [(b * L, L, b * L, L) for b in range(nseq)], -1, -1, 0, 0, mask.reshape(-1) if masked else None, D ** -0.5, do,
                     drop, dtype)
    for name, value in got.items():
        O.check(value, want[name], name)


@pytest.mark.parametrize("nseq,L,H,D,masked,dropout", SDPA)
def test_sdpa_node(nseq, L, H, D, masked, dropout):
    prev = backend.use(RefBackend())
    try:
        sdpa_case("cpu", torch.float32, nseq, L, H, D, masked, dropout)
    finally:
        backend.use(prev)
