"""A compressed Hugging Face decoder on `model.cobalt_cache` in 8 bits, and on a pool whose pages the sequences share: what every layer's
attention answers, against the definition over what the oracle's cache holds after the same writes, and steps recorded in a graph."""
import numpy as np
import pytest
import torch

from oracle import cache8_ref as R8
from test_gpu_cache8 import Setup
from test_gpu_hf_cache import DEV, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,window,sinks,head_dim,pads,pages,block", [
    (torch.float16, None, 0, 64, None, None, 16), (torch.bfloat16, None, 0, 128, [0, 37, 199], 20, 32), (torch.float16, 50, 4, 64, None, 22, 16),
    (torch.float16, 33, 0, 128, [5, 0, 64], None, 32)])
def test_every_layer_attends_as_defined(monkeypatch, dtype, window, sinks, head_dim, pads, pages, block):
    from cobalt_amd import hf_cache as hf, model as Mo
    calls = {}
    real = hf.cobalt_attention

    def record(module, query, key, value, mask, **kw):
        out, none = real(module, query, key, value, mask, **kw)
        calls.setdefault(key._cobalt_layer.index, []).append([x.detach().cpu() for x in (query, key, value, out)])
        return out, none

    monkeypatch.setattr(hf, "cobalt_attention", record)
    m = _model(dtype, window, head_dim, compress=head_dim == 64)
    batch, steps, g = 3, [200, 1, 5, 1, 13], torch.Generator().manual_seed(2)
    cache = Mo.cobalt_cache(m, batch, 256, page=32, sinks=sinks, bits=8, block=block, pages=pages)
    total = 0
    for n in steps:
        total += n
        mask = None if pads is None else torch.stack([(torch.arange(total) >= p).long() for p in pads]).to(DEV)
        m(torch.randint(0, 512, (batch, n), generator=g).to(DEV), past_key_values=cache, attention_mask=mask)
    seqs = cache.layers[0].sequences
    pads = pads or [0] * batch
    if pages:
        assert seqs.tables.lens.tolist() == [total - p for p in pads]
    assert sorted(calls) == [0, 1] and all(len(c) == len(steps) for c in calls.values())
    for layer in calls.values():
        ref, done = R8.Pool(batch * 8, 2, head_dim, 32, block), 0
        table = np.arange(batch * 8).reshape(batch, 8).tolist()
        for query, key, value, out in layer:
            n, done = query.shape[2], done + query.shape[2]
            s = Setup.__new__(Setup)
            s.heads, s.dim, s.lens, s.ref, s.table = 2, head_dim, [done - p for p in pads], ref, torch.tensor(table)
            s.cut = np.concatenate([[0], np.cumsum(s.lens)]).astype(int)
            new = [min(n, s.lens[b]) for b in range(batch)]
            k, v = (torch.cat([x[b, :, n - new[b]:].transpose(0, 1) for b in range(batch)]).float().numpy() for x in (key, value))
            ref.write(table, s.lens, np.concatenate([[0], np.cumsum(new)]).astype(int).tolist(), k, v)
            s.refresh()
            q, o = (torch.cat([x[b, n - new[b]:] for b in range(batch)]) for x in (query.transpose(1, 2), out))
            s.check(q, o, new, window=window, sinks=sinks if window else 0)
            for b in range(batch):
                assert bool((out[b, :n - new[b]] == 0).all())                          # the padding's own rows


@pytest.mark.parametrize("bits", [4, 8])
def test_steps_in_a_graph_take_pages_as_eager_steps_do(bits):
    from cobalt_amd import model as Mo
    m = _model(torch.float16)
    ids = torch.randint(0, 512, (2, 70), generator=torch.Generator().manual_seed(4)).to(DEV)
    mask = torch.ones_like(ids)
    mask[1, :9] = 0
    runs = []
    for recorded in (False, True):
        cache = Mo.cobalt_cache(m, 2, 192, page=16, bits=bits, pages=14)
        seqs = cache.layers[0].sequences
        tok = m(ids, past_key_values=cache, attention_mask=mask).logits[:, -1:].argmax(-1)
        logits = torch.empty(2, 1, 512, dtype=torch.float16, device=DEV)

        def step():
            logits.copy_(m(tok, past_key_values=cache).logits)
            tok.copy_(logits.argmax(-1))

        got = []
        if recorded:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(2):
                    step()
                    got.append((tok.clone(), logits.clone()))
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        for i in range(len(got), 40):
            graph.replay() if recorded else step()
            got.append((tok.clone(), logits.clone()))
            if i % 10 == 9:
                torch.cuda.synchronize()
                torch.empty(1 << 20, dtype=torch.uint8, device=DEV).fill_(255)
        assert int(cache.get_seq_length()) == 110 and seqs.lens.tolist() == [110, 101] == seqs.tables.lens.tolist()
        assert int(seqs.tables.count) == 0
        if recorded:                                                    # replays that the pages do not last for: tokens without a page
            for _ in range(3):
                graph.replay()
            torch.cuda.synchronize()
            assert seqs.lens.tolist() == [113, 104] and seqs.tables.lens.tolist() == [112, 104]
        else:
            with pytest.raises(ValueError, match="14 pages"):
                m(ids[:, :3], past_key_values=cache)
        runs.append(got)
    for i, (a, b) in enumerate(zip(*runs)):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), i


@pytest.mark.parametrize("pages", [None, 8])
def test_generate_runs_and_the_cache_is_reused(pages):
    from cobalt_amd import model as Mo
    m = _model(torch.bfloat16)
    ids = torch.randint(0, 512, (2, 40), generator=torch.Generator().manual_seed(4)).to(DEV)
    cache = Mo.cobalt_cache(m, 2, 100, page=16, bits=8, pages=pages)
    kw = dict(attention_mask=torch.ones_like(ids), max_new_tokens=20, do_sample=False)
    first = m.generate(ids, past_key_values=cache, **kw)
    cache.reset()
    assert first.shape == (2, 60) and torch.equal(m.generate(ids, past_key_values=cache, **kw), first)
    own = Mo.cobalt_cache(m, 2, 100, page=16, bits=8)                   # whose pages they are changes nothing
    assert torch.equal(m.generate(ids, past_key_values=own, **kw), first)
