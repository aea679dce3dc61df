"""The cache object's host side where sequences of a batch take different numbers of tokens:
bounds, pages and refusals.  No GPU: the store itself is left out."""
import pytest
import torch

import monarch_attention_b200 as mab


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(mab.kv_cache, "kv_cache_write", lambda *a, **kw: None)

    def make(num_pages, max_seqs, max_len, page_size=4):
        return mab.PagedKVCache(num_pages, 1, 8, max_seqs=max_seqs, max_len=max_len,
                                page_size=page_size, device="cpu")
    return make


def tokens(c, T):
    x = torch.zeros(len(c.lengths), 1, T, 8, dtype=torch.bfloat16)
    return x, x


@pytest.mark.parametrize("as_tensor", [False, True])
def test_an_idle_sequence_outlives_max_len_steps(cache, as_tensor):
    c = cache(16, 2, 32)
    for step in range(100):
        n = [1 if step < 12 else 0, 0]
        c.append(*tokens(c, 1), count=torch.tensor(n) if as_tensor else n)
    assert c.lengths.tolist() == [12, 0] and c.free_pages == 16 - 3
    assert (c.page_table[1] == -1).all()
    for _ in range(20):  # and the other one still has all of max_len
        c.append(*tokens(c, 1), count=[1, 0])
    with pytest.raises(ValueError, match="33 tokens exceeds max_len"):
        c.append(*tokens(c, 1), count=[1, 0])
    c.append(*tokens(c, 1), count=[0, 1])
    assert c.lengths.tolist() == [32, 1] and c.free_pages == 16 - 9


def test_prompts_of_different_lengths(cache):
    c = cache(16, 2, 32)
    c.append(*tokens(c, 30), count=[30, 2])
    assert c.free_pages == 16 - 8 - 1
    for _ in range(2):
        c.append(*tokens(c, 1))
    with pytest.raises(ValueError, match="33 tokens"):
        c.append(*tokens(c, 1))
    assert c.lengths.tolist() == [32, 4] and c._bound == [32, 4]
    c.free(0)
    c.append(*tokens(c, 1))
    assert c.lengths.tolist() == [1, 5] and c.free_pages == 16 - 1 - 2


def test_counts_are_clamped_and_checked(cache):
    c = cache(16, 3, 32)
    c.append(*tokens(c, 5), count=[9, -3, 5])
    assert c.lengths.tolist() == [5, 0, 5] and c._bound == [5, 0, 5]
    with pytest.raises(ValueError, match="3 entries; got 2"):
        c.append(*tokens(c, 1), count=[1, 1])
    with pytest.raises(TypeError):
        c.append(*tokens(c, 1), count=[0.5, 1, 1])
    with pytest.raises(TypeError):
        c.append(*tokens(c, 1), count=torch.tensor([0.5, 1, 1]))
    assert c.lengths.tolist() == [5, 0, 5] and c._bound == [5, 0, 5] and c.free_pages == 12


def test_a_full_pool_is_full_for_those_that_take(cache):
    c = cache(3, 3, 32)
    c.append(*tokens(c, 8), count=[8, 4, 0])
    assert c.free_pages == 0
    for _ in range(3):
        c.append(*tokens(c, 1), count=[0, 0, 0])
    with pytest.raises(RuntimeError, match="full: 1 pages wanted, 0 free"):
        c.append(*tokens(c, 1), count=[0, 0, 1])
    c.free(1)
    c.append(*tokens(c, 1), count=[0, 0, 1])
    assert c.lengths.tolist() == [8, 0, 1]


def test_tighten_takes_the_lengths_and_keeps_what_is_reserved(cache):
    c = cache(16, 2, 32)
    c.append(*tokens(c, 20))
    c.reserve([4, 28])
    assert c.free_pages == 16 - 5 - 7
    c.lengths.copy_(torch.tensor([6, 3]))  # as a captured graph leaves them
    before = c.page_table.clone()
    c.tighten()
    assert c._bound == [6, 3] and c.free_pages == 16 - 2 - 7
    assert torch.equal(c.page_table[0, :2], before[0, :2]) and (c.page_table[0, 2:] == -1).all()
    assert torch.equal(c.page_table[1], before[1])
    c.reserve([32, 32])
    ids = c.page_table[c.page_table >= 0].tolist()
    assert len(ids) == len(set(ids)) == 16 and c.free_pages == 0
    for e in range(2):
        c.free(e)
    assert c.free_pages == 16 and c._reserved == [0, 0]
