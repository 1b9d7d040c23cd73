"""One workspace that serves several kinds of paged reads in turn."""

import pytest
import torch

from tests.paged_reference import assert_within, make_cache, page_table, sm_scale
from tests.test_gpu_paged_read import reference


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (32, 8, 64), (8, 2, 256)])
@pytest.mark.parametrize("made", ["attend_workspace", "large"])
def test_one_workspace_serves_every_read_in_turn(kind, hq, hkv, d, made):
    """A model with full and sliding layers over one cache: reads without options (which keep tickets at the head of the
    workspace, zero between calls), reads with a window and prefills, all on one workspace."""
    from bpt_b200.kernels.kv_attention import attend, attend_workspace, paged_split
    from bpt_b200.kernels.prefill_attention import prefill_attend

    g = torch.Generator().manual_seed(hq)
    lengths = [10, 0] + torch.randint(300, 1500, (30,), generator=g).tolist()  # (sequences in a few parts each)
    batch = len(lengths)
    table, blocks = page_table(lengths, 16, g)
    kv, keys, values = make_cache(kind, blocks, 16, hkv, d, table, g)
    split = paged_split(batch, max(lengths))
    if made == "large":
        ws = torch.zeros(128 << 20, dtype=torch.uint8, device="cuda")
    else:
        ws = attend_workspace(batch, hq, d, -(-max(lengths) // split), torch.device("cuda", 0)).clone()
    n, cu = torch.tensor(lengths, dtype=torch.int32).cuda(), torch.arange(batch + 1, dtype=torch.int32).cuda()
    vmax = values.abs().max().item()
    for _ in range(2):
        for read in ("full", "sliding", "full", "prefill", "full"):
            q = torch.randn(batch, hq, d, generator=g).to(torch.bfloat16)
            out = torch.full((batch, hq, d), float("nan"), device="cuda")
            if read == "prefill":  # one new token each
                if made == "large":
                    out = prefill_attend(q.cuda(), kv, cu, n, sm_scale(d), workspace=ws)
            else:
                attend(q.cuda(), kv, n, sm_scale(d), window=500 if read == "sliding" else 0, out=out, workspace=ws)
            if read != "prefill" or made == "large":
                want = reference(q, keys, values, table, lengths, 16, window=500 if read == "sliding" else 0)
                # 8-bit keys and values are the operands themselves; queries and probabilities have 11 bits at least
                assert_within(out, want, out.dtype, vmax, 11)
            ws[256 << 10 :].fill_(255)  # what follows the tickets may hold anything: here NaN
