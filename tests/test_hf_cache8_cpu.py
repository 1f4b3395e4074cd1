"""A Hugging Face decoder on the 8-bit cache and on a pool whose pages the sequences share, without the GPU: the operators are replaced by exact
ones, and the tables by the oracle's, as in the tests of the 4-bit cache."""
import pytest
import torch

from cobalt_amd import KVCache, KVCache8, KVRows
from oracle import cache8_ref as R8
from test_hf_cache_cpu import ATOL, Mo, _model, exact, hf, tr  # noqa: F401


@pytest.fixture
def tables(exact, monkeypatch):
    """ops.cache_pages by the oracle, one page after the other, on the arrays of the KVPages"""
    calls = []

    def cache_pages(pool, lens, starts=None):
        t = R8.Tables(pool.pages, pool.seqs, pool.max_len, pool.page)
        t.table, t.lens, t.free, t.count = pool.table.tolist(), pool.lens.tolist(), pool.free.tolist(), int(pool.count)
        starts = t.resize(lens.tolist())
        for x, y in ((pool.table, t.table), (pool.lens, t.lens), (pool.free, t.free), (pool.count, [t.count])):
            x.copy_(torch.tensor(y, dtype=torch.int32))
        calls.append(lens.tolist())
        return KVRows(pool.table, pool.lens, torch.tensor(starts, dtype=torch.int32))

    monkeypatch.setattr(hf.ops, "cache_pages", cache_pages)
    return calls


def _steps(cache, m, steps, pads):
    g = torch.Generator().manual_seed(5)
    want = tr.DynamicCache(config=m.config)
    total = 0
    for n in steps:
        ids = torch.randint(2, 97, (len(pads), n), generator=g)
        total += n
        mask = torch.stack([(torch.arange(total) >= p).long() for p in pads])
        with torch.no_grad():
            m.set_attn_implementation("sdpa")
            a = m(ids, past_key_values=want, attention_mask=mask).logits
            m.set_attn_implementation(hf.NAME)
            b = m(ids, past_key_values=cache, attention_mask=mask).logits
        for i, p in enumerate(pads):
            first = max(0, p - (total - n))
            assert float((a[i, first:] - b[i, first:]).abs().max()) < ATOL


@pytest.mark.parametrize("pads", [[0, 0, 0], [0, 19, 5]])
@pytest.mark.parametrize("bits", [4, 8])
def test_sequences_that_share_a_pool(tables, bits, pads):
    m = _model()
    cache = Mo.cobalt_cache(m, 3, 200, page=16, bits=bits, pages=12)
    seqs = cache.layers[0].sequences
    for _ in range(2):
        _steps(cache, m, [30, 1, 5, 1, 11], pads)                       # three pages each: nine of twelve
        assert isinstance(cache.layers[0].pool, KVCache if bits == 4 else KVCache8) and cache.layers[0].pool.pages == 12
        need = sum(-(-(48 - p) // 16) for p in pads)
        assert seqs.lens.tolist() == [48 - p for p in pads] == seqs.tables.lens.tolist() and int(seqs.tables.count) == 12 - need
        with pytest.raises(ValueError, match="pages of 16 tokens, the step ends with"):
            m(torch.ones(3, 40, dtype=torch.long), past_key_values=cache)
        assert seqs.lens.tolist() == [48 - p for p in pads]
        cache.reset()
        assert int(seqs.tables.count) == 12 and bool((seqs.table == -1).all())


def test_a_first_step_that_the_pages_do_not_last_for(tables):
    m = _model()
    cache = Mo.cobalt_cache(m, 2, 100, page=16, pages=3)
    with pytest.raises(ValueError, match="3 pages"):
        m(torch.ones(2, 20, dtype=torch.long), past_key_values=cache)
    m(torch.ones(2, 20, dtype=torch.long), past_key_values=cache, attention_mask=torch.tensor([[1] * 20, [0] * 4 + [1] * 16]))
    assert cache.layers[0].sequences.tables.lens.tolist() == [20, 16]


def test_pages_that_replays_take_go_back(tables, monkeypatch):
    m = _model()
    recording = [False]
    monkeypatch.setattr(hf, "_recording", lambda: recording[0], raising=False)
    cache = Mo.cobalt_cache(m, 1, 64, page=16, pages=4)
    seqs = cache.layers[0].sequences
    m(torch.ones(1, 16, dtype=torch.long), past_key_values=cache)
    recording[0] = True
    m(torch.ones(1, 1, dtype=torch.long), past_key_values=cache)
    recording[0] = False
    assert int(seqs.tables.count) == 2
    cache.reset()
    assert int(seqs.tables.count) == 4


def test_refusals():
    m = _model()
    with pytest.raises(ValueError, match="4 or 8 bits"):
        Mo.cobalt_cache(m, 1, 64, bits=6)
    with pytest.raises(ValueError):
        Mo.cobalt_cache(m, 1, 64, pages=0)
    cache = Mo.cobalt_cache(m, 1, 64, page=16, bits=8, block=32)
    k = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="block"):
        cache.layers[0].lazy_initialization(k, k)
