"""A compressed Hugging Face decoder on `model.cobalt_cache`: what every layer's attention answers, against the definition in
float64 over the layer's own keys and values (bounds as for the operators themselves), and steps recorded in a graph."""
import numpy as np
import pytest
import torch

from oracle import cache_ref as R
from test_gpu_cache import Setup

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _model(dtype, window=None, head_dim=64, compress=True):
    tr = pytest.importorskip("transformers")
    from cobalt_amd import model as Mo
    cfg = tr.MistralConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                           num_key_value_heads=2, head_dim=head_dim, max_position_embeddings=1024, sliding_window=window, eos_token_id=None,
                           attn_implementation="sdpa")
    torch.manual_seed(0)
    m = tr.MistralForCausalLM(cfg).to(DEV, dtype).eval().requires_grad_(False)
    if compress:
        Mo.compress_model(m, None, sparsity=0.5, bits=4, group=128)
    return m


@pytest.mark.parametrize("dtype,window,sinks,head_dim,pads", [
    (torch.float16, None, 0, 64, None), (torch.bfloat16, None, 0, 128, [0, 37, 199]), (torch.float16, 50, 4, 64, None),
    (torch.float16, 33, 0, 128, [5, 0, 64])])
def test_every_layer_attends_as_defined(monkeypatch, dtype, window, sinks, head_dim, pads):
    from cobalt_amd import hf_cache as hf, model as Mo
    calls = {}
    real = hf.cobalt_attention

    def record(module, query, key, value, mask, **kw):
        out, none = real(module, query, key, value, mask, **kw)
        calls.setdefault(key._cobalt_layer.index, []).append([x.detach().cpu() for x in (query, key, value, out)])
        return out, none

    monkeypatch.setattr(hf, "cobalt_attention", record)
    m = _model(dtype, window, head_dim, compress=head_dim == 64)
    batch, steps, g = 3, [200, 1, 5, 1], torch.Generator().manual_seed(2)
    cache = Mo.cobalt_cache(m, batch, 256, page=32, sinks=sinks)
    total = 0
    for n in steps:
        total += n
        mask = None if pads is None else torch.stack([(torch.arange(total) >= p).long() for p in pads]).to(DEV)
        m(torch.randint(0, 512, (batch, n), generator=g).to(DEV), past_key_values=cache, attention_mask=mask)
    pads = pads or [0] * batch
    assert sorted(calls) == [0, 1] and all(len(c) == len(steps) for c in calls.values())
    for layer in calls.values():
        done = 0
        for query, key, value, out in layer:
            n, done = query.shape[2], done + query.shape[2]
            s = Setup.__new__(Setup)
            s.heads, s.dim, s.lens = 2, head_dim, [done - p for p in pads]
            s.cut = np.concatenate([[0], np.cumsum(s.lens)]).astype(int)
            past = [torch.cat([c[i] for c in layer], 2) for i in (1, 2)]                 # [batch, heads, tokens, dim]
            k, v = (torch.cat([x[b, :, pads[b]:done].transpose(0, 1) for b in range(batch)]).float().numpy() for x in past)
            s.hk, s.hv = R.held(k, v, 32)
            new = [min(n, s.lens[b]) for b in range(batch)]
            q, o = (torch.cat([x[b, n - new[b]:] for b in range(batch)]) for x in (query.transpose(1, 2), out))
            s.check(q, o, new, window=window, sinks=sinks if window else 0)
            for b in range(batch):
                assert bool((out[b, :n - new[b]] == 0).all())                          # the padding's own rows


def test_steps_in_a_graph_answer_as_eager_steps():
    from cobalt_amd import model as Mo
    m = _model(torch.float16)
    ids = torch.randint(0, 512, (2, 70), generator=torch.Generator().manual_seed(4)).to(DEV)
    mask = torch.ones_like(ids)
    mask[1, :9] = 0
    runs = []
    for recorded in (False, True):
        cache = Mo.cobalt_cache(m, 2, 192)
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
        assert int(cache.get_seq_length()) == 110 and cache.layers[0].sequences.lens.tolist() == [110, 101]
        runs.append(got)
    for i, (a, b) in enumerate(zip(*runs)):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), i


def test_recording_refuses_what_needs_the_host():
    from cobalt_amd import model as Mo
    m = _model(torch.float16, compress=False)
    tok = torch.zeros(1, 1, dtype=torch.long, device=DEV)
    cache = Mo.cobalt_cache(m, 1, 64)
    layer = cache.layers[0]
    k = torch.zeros(1, 2, 1, 64, dtype=torch.float16, device=DEV)
    mask = torch.ones(1, 1, dtype=torch.long, device=DEV)
    m(tok, past_key_values=Mo.cobalt_cache(m, 1, 64))                   # libraries start outside the recording
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        k.add_(1)
        with pytest.raises(RuntimeError, match="recorded in a graph"):
            layer.update(k, k)
        with pytest.raises(ValueError, match="recorded in a graph"):
            layer.sequences.begin(1, 1, mask)
    assert layer.pool is None and int(cache.get_seq_length()) == 0


def test_generate_runs_and_the_cache_is_reused():
    from cobalt_amd import model as Mo
    m = _model(torch.bfloat16)
    ids = torch.randint(0, 512, (2, 40), generator=torch.Generator().manual_seed(4)).to(DEV)
    cache = Mo.cobalt_cache(m, 2, 100)
    kw = dict(attention_mask=torch.ones_like(ids), max_new_tokens=20, do_sample=False)
    first = m.generate(ids, past_key_values=cache, **kw)
    cache.reset()
    assert first.shape == (2, 60) and torch.equal(m.generate(ids, past_key_values=cache, **kw), first)


def test_eager_steps_after_replays():
    from cobalt_amd import model as Mo
    m = _model(torch.float16)
    ids = torch.randint(0, 512, (2, 60), generator=torch.Generator().manual_seed(4)).to(DEV)
    mask = lambda n: torch.stack([(torch.arange(n) >= p).long() for p in (0, 9)]).to(DEV)
    runs = []
    for recorded in (False, True):
        cache = Mo.cobalt_cache(m, 2, 64)
        got = [m(ids[:, :40], past_key_values=cache, attention_mask=mask(40)).logits]
        tok = ids[:, 40:41].clone()
        if recorded:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got.append(m(tok, past_key_values=cache).logits.clone())
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = m(tok, past_key_values=cache).logits
        else:
            got.append(m(tok, past_key_values=cache).logits)
        for i in range(41, 50):
            tok.copy_(ids[:, i:i + 1])
            if recorded:
                graph.replay()
                got.append(out.clone())
            else:
                got.append(m(tok, past_key_values=cache).logits)
        got.append(m(ids[:, 50:51], past_key_values=cache, attention_mask=mask(51)).logits)     # as generate passes it
        got.append(m(ids[:, 51:60], past_key_values=cache).logits)
        assert int(cache.get_seq_length()) == 60 and cache.layers[0].sequences.lens.tolist() == [60, 51]
        with pytest.raises(ValueError, match="for 64 tokens"):
            m(ids[:, :5], past_key_values=cache)
        runs.append(got)
    for i, (a, b) in enumerate(zip(*runs)):
        assert torch.equal(a, b), i
