"""prefill_attend launched with programmatic dependent launch before another kernel that takes tensor memory."""

from pathlib import Path

import pytest
import torch

from tests.paged_reference import sm_scale
from tests.test_gpu_paged_prefill import case

CSRC = Path(__file__).resolve().parents[1] / "bytes-per-token_b200" / "csrc"


@pytest.mark.parametrize("source", ["paged_prefill_tc.cu", "w4a16_tc.cu"])
def test_dependents_start_behind_the_allocation(source):
    """A dependent CTA that took tensor memory which a CTA of this grid still needs would wait for this grid, and this grid
    for the memory: every CTA allocates before it lets dependents start."""
    text = (CSRC / source).read_text()
    assert text.count("pdl_launch_dependents();") == 1 and text.count("tcgen05.alloc.") == 1
    assert text.index("tcgen05.alloc.") < text.index("pdl_launch_dependents();")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 64), (16, 4, 128), (8, 8, 256)])
@pytest.mark.parametrize("seqs", [[(0, 700), (33, 200)], [(3000, 20)]], ids=["tiles", "parts"])
def test_prefill_then_a_dependent_linear(kind, hq, hkv, d, seqs):
    """A layer's order: attention, then its output projection (tcgen05 at 16 tokens and more), each let in early by the kernel
    before it, equals the same calls in plain stream order."""
    from bpt_b200 import _lib
    from bpt_b200.kernels.prefill_attention import prefill_attend
    from bpt_b200.kernels.w4a16 import quantize_w4a16, w4a16_linear

    kv, _, _, q, _, cu, lengths = case(kind, seqs, hq, hkv, d, 16, seed=d, q_dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(1)
    weight = quantize_w4a16((torch.randn(2048, hq * d, generator=g, device="cuda") * 0.02).to(torch.bfloat16), 128)
    args = (q.cuda(), kv, cu.cuda(), lengths.cuda(), sm_scale(d))
    want = w4a16_linear(prefill_attend(*args).flatten(1), *weight, group=128)
    for _ in range(3):
        for _ in range(8):
            got = w4a16_linear(prefill_attend(*args, pdl=True).flatten(1), *weight, group=128, pdl=True)
        assert torch.equal(got, want)
    assert _lib.device_error() == 0
