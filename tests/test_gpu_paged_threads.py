"""The workspaces that the paged reads take by themselves, under two threads on one stream."""

import threading

import pytest
import torch

from tests.paged_reference import make_cache, page_table


@pytest.mark.gpu
def test_threads_on_one_stream_do_not_share_a_workspace():
    """A read is two launches that pass its parts through a workspace: another thread's launches may come between them."""
    from bpt_b200.kernels.kv_attention import _scratch, attend
    from bpt_b200.kernels.prefill_attention import prefill_attend

    device, calls = torch.device("cuda", 0), []
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        table, blocks = page_table([4000, 900], 16, g)
        kv, _, _ = make_cache("bf16", blocks, 16, 4, 64, table, g)
        q = torch.randn(2, 8, 64, generator=g).to(torch.bfloat16).cuda()
        n, cu = torch.tensor([4000, 900], dtype=torch.int32).cuda(), torch.arange(3, dtype=torch.int32).cuda()
        calls.append((q, kv, n, cu, attend(q, kv, n, 0.125), prefill_attend(q, kv, cu, n, 0.125)))
    torch.cuda.synchronize()
    together, found = threading.Barrier(2), [None, None]

    def work(i):
        q, kv, n, cu, decoded, prefilled = calls[i]
        mine = _scratch(1 << 20, device)
        wrong = torch.zeros((), dtype=torch.int64, device="cuda")
        together.wait()
        for _ in range(300):
            wrong += (attend(q, kv, n, 0.125) != decoded).sum() + (prefill_attend(q, kv, cu, n, 0.125) != prefilled).sum()
        torch.cuda.synchronize()
        found[i] = (int(wrong), mine.data_ptr())
        together.wait()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert found[0][1] != found[1][1]
    assert found[0][0] == 0 and found[1][0] == 0
