"""Bookkeeping of PagedKVCache on the host: pages, slots, lengths, what is
refused, and pages freed behind a window."""
import numpy as np
import pytest
import torch

from walsh_research_b200.model import PagedKVCache


def make(**kw):
    d = dict(n_layers=2, n_pages=10, page_size=4, n_head=2, head_dim=16, device="cpu", dtype=torch.float16, max_seqs=3,
             max_seq_len=24)
    d.update(kw)
    return PagedKVCache(**d)


def owned(c):
    return sorted(c._table[c._table >= 0].tolist())


def test_steps_lay_out_every_token_in_its_own_slot():
    c = make()
    a, b = c.add(2)
    s = c.select([a]).begin(6)
    assert s.positions.tolist() == list(range(6)) and s.kv_lens.tolist() == [6] and s.q_offsets.tolist() == [0, 6]
    c.select([a]).increment(6)
    batch = c.select([b, a])
    s = batch.begin(3)
    assert s.positions.tolist() == [0, 1, 2, 6, 7, 8] and s.kv_lens.tolist() == [3, 9] and s.max_len == 9
    assert s.q_offsets.tolist() == [0, 3, 6] and s.page_table.shape == (2, 3)
    for i, (seq, pos) in enumerate(zip([b] * 3 + [a] * 3, s.positions.tolist())):
        row = [b, a].index(seq)
        assert int(s.slots[i]) == int(s.page_table[row, pos // 4]) * 4 + pos % 4
    assert len(set(s.slots.tolist())) == 6
    batch.increment(3)
    assert c.lengths([a, b]) == [9, 3]
    assert len(owned(c)) == 4 and len(set(owned(c))) == 4 and c.free_pages == 6
    c.remove([a])
    assert c.free_pages == 9 and c.lengths([b]) == [3]
    assert c.add(2) and c.lengths([b]) == [3]


def test_out_of_pages_changes_nothing():
    c = make(n_pages=3)
    a, b = c.add(2)
    c.select([a]).begin(8)
    c.select([a]).increment(8)
    with pytest.raises(RuntimeError, match="out of pages"):
        c.select([a, b]).begin(4)
    assert c.free_pages == 1 and c.lengths([a, b]) == [8, 0] and (c._table[b] < 0).all()
    c.select([b]).begin(4)
    assert c.free_pages == 0


def test_refusals():
    c = make()
    (a,) = c.add()
    for bad in ([a, a], [a + 1], [-1], [99]):
        with pytest.raises(ValueError):
            c.select(bad)
    with pytest.raises(RuntimeError):
        c.add(3)
    with pytest.raises(ValueError, match="per sequence"):
        c.select([a]).begin(25)
    c.remove([a])
    with pytest.raises(ValueError):
        c.select([a])
    for kw in (dict(n_pages=0), dict(page_size=0), dict(window=-1), dict(max_seqs=0)):
        with pytest.raises(ValueError):
            make(**kw)


@pytest.mark.parametrize("window,sinks", [(5, 0), (5, 3), (4, 4), (1, 0), (9, 5)])
def test_pages_behind_the_window_are_freed_and_no_visible_key_is(window, sinks):
    c = make(n_pages=24, max_seq_len=96, window=window, sinks=sinks)
    (a,) = c.add()
    for n in [7] + [1] * 60:
        c.select([a]).begin(n)
        pos0 = c.lengths([a])[0]
        for p in range(pos0, pos0 + n):
            for key in range(p + 1):
                if key > p - window or key < sinks:
                    assert c._table[a, key // 4] >= 0, (p, key)
        c.select([a]).increment(n)
    pages = owned(c)
    assert len(set(pages)) == len(pages) and len(pages) + c.free_pages == 24
    assert len(pages) <= -(-sinks // 4) + -(-window // 4) + 1


def test_table_rows_are_free_of_other_sequences():
    rng = np.random.default_rng(0)
    c = make(n_pages=40, max_seqs=6)
    live = []
    for _ in range(300):
        if live and rng.random() < 0.3:
            c.remove([live.pop(int(rng.integers(len(live))))])
        elif len(live) < 6:
            live += c.add()
        if live and c.lengths(live) and max(c.lengths(live)) < 20:
            c.select(live).begin(2)
            c.select(live).increment(2)
        assert len(set(owned(c))) == len(owned(c)) == 40 - c.free_pages


def test_batches_of_nothing_or_of_removed_sequences_are_refused():
    c = make()
    a, b = c.add(2)
    batch = c.select([a, b])
    for what in (lambda: c.select([]).begin(1), lambda: batch.begin(0), lambda: batch.increment(-1)):
        with pytest.raises(ValueError):
            what()
    batch.begin(3)
    batch.increment(3)
    c.remove([a])
    for what in (lambda: batch.begin(1), lambda: batch.increment(1)):
        with pytest.raises(ValueError):
            what()
    assert c.free_pages == 9 and c.lengths([b]) == [3]


def test_a_batch_of_a_removed_sequence_is_refused_although_its_row_is_in_use_again():
    c = make()
    a = c.add()
    old = c.select(a)
    c.remove(a)
    b = c.add()
    assert a == b                                          # the row is handed out again
    for call in (lambda: old.begin(2), lambda: old.increment(2)):
        with pytest.raises(ValueError, match="removed"):
            call()
    assert c.lengths(b) == [0] and c.free_pages == 10
    new = c.select(b)
    new.begin(2)
    new.increment(2)
    assert c.lengths(b) == [2]


def test_a_forward_that_is_refused_reserves_nothing():
    """Positions past the rotation table, a batch of another size or type, start positions."""
    from walsh_research_b200.model import mHCWalsh
    c = make()
    (a,) = c.add()
    c.select([a]).begin(6)
    c.select([a]).increment(6)
    batch = c.select([a])
    for args in ((1, 7, 0, torch.float16, 12), (2, 7, 0, torch.float16, 24), (1, 7, 0, torch.float32, 24),
                 (1, 7, 3, torch.float16, 24), (1, 19, 0, torch.float16, 30)):
        with pytest.raises(ValueError):
            mHCWalsh._begin_paged(batch, *args)
        assert c.free_pages == 8 and c.lengths([a]) == [6]
    assert mHCWalsh._begin_paged(batch, 1, 7, 0, torch.float16, 13).max_len == 13 and c.free_pages == 6
