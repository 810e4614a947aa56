"""What the kernels report through a paged cache reaches the caller."""
import pytest
import torch

import test_gpu_paged_model as P
from walsh_research_b200.model import paged

pytestmark = pytest.mark.gpu


def test_generate_batch_raises_what_a_kernel_reported(monkeypatch):
    """A slot past the pool (as a wrong page table would give) is skipped and reported by the append kernel."""
    cfg, _, _, m = P._model()
    prompts = [P._ids(cfg, t, seed=t) for t in (3, 5)]
    begin = paged.PagedBatch.begin
    m.generate_batch(prompts, 3, top_k=1)

    def wrong(self, n):
        step = begin(self, n)
        step.slots[-1] = self.cache.n_pages * self.cache.page_size
        return step

    monkeypatch.setattr(paged.PagedBatch, "begin", wrong)
    with pytest.raises(IndexError, match="out of range"):
        m.generate_batch(prompts, 3, top_k=1)
    monkeypatch.undo()
    assert torch.equal(m.generate_batch(prompts, 3, top_k=1)[0][:3], prompts[0])


def test_a_cache_stays_on_the_device_it_was_made_on():
    """"cuda" is the device that is current at construction, not at each call."""
    c = paged.PagedKVCache(1, 4, 4, 2, 16, "cuda", max_seqs=1, max_seq_len=8)
    assert c.device == c.k_pages[0].device and c.device.index is not None
    step = c.select(c.add()).begin(3)
    assert step.slots.device == step.page_table.device == c.k_pages[0].device
