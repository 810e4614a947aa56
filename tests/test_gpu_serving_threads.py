"""Serving entry points called from several host threads at once, each on a stream of its own."""
import threading

import pytest
import torch

from walsh_research_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_sampling_of_different_vocabularies_in_several_threads():
    """Rows are held in shared memory, of an amount that depends on the
    vocabulary; the C entry is called in tight loops, so that calls overlap."""
    fn, failed = _lib.lib().walsh_sample_tokens, []

    def work(vocab):
        rows = 150
        g = torch.Generator(device=DEV).manual_seed(vocab)
        z, u = torch.randn(rows, vocab, generator=g, device=DEV), torch.rand(rows, generator=g, device=DEV)
        ids = torch.empty(rows, dtype=torch.int64, device=DEV)
        want = ops.sample_tokens(z, u, top_k=5)
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()) as _:
            s = torch.cuda.current_stream()
            args = (z.data_ptr(), _lib.F32, vocab, rows, vocab, u.data_ptr(), 1.0, 5, 1.0, 0.0, None, None, None, None,
                    ids.data_ptr(), None, s.cuda_stream)
            start.wait()
            codes = {fn(*args) for _ in range(3000)}
            s.synchronize()
        if codes != {0} or not torch.equal(ids, want):
            failed.append((vocab, codes))

    vocabs = [24000, 3000, 12000, 5000]
    start = threading.Barrier(len(vocabs))
    threads = [threading.Thread(target=work, args=(v,)) for v in vocabs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
