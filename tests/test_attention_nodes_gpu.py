"""Autograd nodes of the text tower's attention on the device: values and gradients against the 64-bit form."""
import pytest
import torch

from tests.test_attention_nodes_cpu import SDPA, sdpa_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nseq,L,H,D,masked,dropout", SDPA)
def test_sdpa_node(nseq, L, H, D, masked, dropout, dtype):
    """The kernels round what the bounds count: P, dS and the results to the operand type, scores and sums in f32."""
    sdpa_case("cuda", dtype, nseq, L, H, D, masked, dropout)
