"""The serving operators called by several host threads at once, each on its own stream and workspace."""
from __future__ import annotations

import threading

import pytest

from test_serving_operators_gpu import Paged, check_attention

pytestmark = pytest.mark.gpu


def test_threads_with_their_own_streams(cuda):
    import torch
    heads, kinds = 28, [[(1, 3000), (1, 50)], [(90, 2000), (1, 700)], [(4, 900)], [(300, 300), (64, 64)]]
    jobs, errors = [], []
    for seed, sequences in enumerate(kinds):
        paged = Paged(cuda, sequences, 4, 128, 16, ("fp16", "bf16")[seed % 2], seed=seed)
        q = torch.randn(paged.tokens, heads * 128, generator=paged.generator, device=cuda).to(paged.dtype)
        out, lse = torch.empty_like(q), torch.empty(paged.tokens, heads, device=cuda)
        jobs.append((paged, q, out, lse, torch.cuda.Stream(), torch.empty(64 << 20, dtype=torch.uint8, device=cuda)))
    torch.cuda.synchronize()
    start = threading.Barrier(len(jobs))

    def work(paged, q, out, lse, stream, workspace):
        try:
            torch.cuda.set_device(cuda)
            start.wait()
            for _ in range(50):
                paged.attention(q, heads, out, lse, workspace=workspace, stream=stream.cuda_stream)
        except Exception as error:  # noqa: BLE001  (reported by the test's own thread)
            errors.append(error)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for paged, q, out, lse, *_ in jobs:
        assert int(paged.status) == 0
        check_attention(paged, q, out, lse, heads)
