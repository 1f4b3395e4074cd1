"""A Hugging Face decoder on `model.cobalt_cache`, without the GPU: the two operators are replaced by exact ones (nothing rounded,
float64), so the logits must be those of the same float64 model with its own attention and cache: which rows, lengths, windows,
padding and positions the decoder hands to the operators.  The five norms of the model round to float32 whatever its type, so sums in
another order may come out half a step apart there, 2^-23 relative: 1e-5 is 80 such steps of values around 1, a wrong row or mask is above 1e-2."""
import numpy as np
import pytest
import torch

from oracle import cache_ref as R

tr = pytest.importorskip("transformers")
Mo = pytest.importorskip("cobalt_amd.model")
hf = pytest.importorskip("cobalt_amd.hf_cache")
ATOL = 1e-5


def _model(window=None, layers=2):
    cfg = tr.MistralConfig(vocab_size=97, hidden_size=128, intermediate_size=128, num_hidden_layers=layers, num_attention_heads=4,
                           num_key_value_heads=2, head_dim=64, max_position_embeddings=512, sliding_window=window, pad_token_id=0,
                           bos_token_id=1, eos_token_id=None, attn_implementation="sdpa")
    torch.manual_seed(3)
    return tr.MistralForCausalLM(cfg).double().eval().requires_grad_(False)


def _tokens(rows, seqs, tokens):
    """(row, sequence, token) of every row of a call that belongs to a sequence."""
    starts = (torch.arange(seqs + 1) * (tokens // seqs) if rows.starts is None else rows.starts).tolist()
    for b, n in enumerate(rows.lens.tolist()):
        for r in range(starts[b], starts[b + 1]):
            yield r, b, n - (starts[b + 1] - r)


@pytest.fixture
def exact(monkeypatch):
    """The operators with a dense float64 pool in place of the 4-bit one."""
    pools = {}

    def write(cache, k, v, rows):
        pool = pools.setdefault(id(cache), np.full((2, cache.pages * cache.page, cache.heads, cache.head_dim), np.nan))
        for r, b, t in _tokens(rows, rows.lens.numel(), k.shape[0]):
            page = int(rows.table[b, t // cache.page]) if t >= 0 else -1
            if page >= 0:
                pool[:, page * cache.page + t % cache.page] = torch.stack([k[r], v[r]]).numpy()

    def attention(cache, q, rows, scale=None, window=None, sinks=0, out=None):
        out = torch.zeros_like(q)
        ratio = q.shape[1] // cache.heads
        for r, b, t in _tokens(rows, rows.lens.numel(), q.shape[0]):
            pages = rows.table[b].tolist()
            if t < 0 or pages[0] < 0:
                continue
            at = np.array([pages[j // cache.page] * cache.page + j % cache.page for j in range(t + 1)])
            k, v = pools[id(cache)][:, at]
            for h in range(q.shape[1]):
                o = R.attention(q[r:r + 1, h].numpy(), k[:, h // ratio], v[:, h // ratio], np.array([t]), np.ones(t + 1, bool), scale, window, sinks)[0]
                out[r, h] = torch.from_numpy(o[0])
        return out

    monkeypatch.setattr(hf, "DTYPES", (torch.float64,))
    monkeypatch.setattr(hf.ops, "cache_write", write)
    monkeypatch.setattr(hf.ops, "cache_attention", attention)


def _same_steps(window, steps, batch=2, pads=None, page=16):
    m = _model(window)
    g = torch.Generator().manual_seed(5)
    calls = [torch.randint(2, 97, (batch, n), generator=g) for n in steps]
    masks = [None] * len(calls)
    if pads is not None:
        total = 0
        for i, ids in enumerate(calls):
            total += ids.shape[1]
            masks[i] = torch.stack([(torch.arange(total) >= p).long() for p in pads])
    want, dense = [], tr.DynamicCache(config=m.config)
    with torch.no_grad():
        for ids, mask in zip(calls, masks):
            want.append(m(ids, past_key_values=dense, attention_mask=mask).logits)
        cache = Mo.cobalt_cache(m, batch, 128, page=page)
        assert m.config._attn_implementation == "cobalt_cache"
        for i, (ids, mask) in enumerate(zip(calls, masks)):
            got = m(ids, past_key_values=cache, attention_mask=mask).logits
            for b in range(batch):
                first = pads[b] if pads is not None and i == 0 else 0
                assert float((got[b, first:] - want[i][b, first:]).abs().max()) < ATOL, (i, b)
    assert int(cache.get_seq_length()) == sum(steps)
    return m, cache


@pytest.mark.parametrize("window", [None, 7, 2])
def test_prompt_steps_and_drafts_answer_as_the_model_does(exact, window):
    _same_steps(window, [33, 1, 1, 4, 1])


def test_a_batch_padded_in_front(exact):
    _same_steps(None, [20, 1, 1, 3], batch=3, pads=[0, 19, 6])


def test_padding_under_a_window(exact):
    _same_steps(5, [18, 1, 2], batch=2, pads=[11, 0])


def test_a_mask_without_padding_changes_nothing(exact):
    _same_steps(None, [9, 1], batch=2, pads=[0, 0])


def test_generate_answers_as_with_the_models_own_cache(exact):
    m = _model()
    ids = torch.randint(2, 97, (2, 11), generator=torch.Generator().manual_seed(1))
    mask = torch.ones_like(ids)
    mask[1, :4] = 0
    kw = dict(attention_mask=mask, max_new_tokens=9, do_sample=False)
    want = m.generate(ids, **kw)
    cache = Mo.cobalt_cache(m, 2, 64)
    assert torch.equal(m.generate(ids, past_key_values=cache, **kw), want)
    cache.reset()                                                      # an emptied cache takes the next batch, padded otherwise
    mask = torch.ones_like(ids)
    mask[0, :2] = 0
    kw["attention_mask"] = mask
    again = m.generate(ids, past_key_values=cache, **kw)
    m.set_attn_implementation("sdpa")
    assert torch.equal(again, m.generate(ids, **kw))


def test_sinks_reach_the_layers_with_a_window_only(exact, monkeypatch):
    seen = []
    real = hf.ops.cache_attention
    monkeypatch.setattr(hf.ops, "cache_attention", lambda *a, **k: seen.append((k["window"], k["sinks"])) or real(*a, **k))
    ids = torch.arange(2, 12)[None]
    for window, want in ((6, (6, 2)), (None, (None, 0))):
        m = _model(window)
        m(ids, past_key_values=Mo.cobalt_cache(m, 1, 32, sinks=2))
        assert set(seen) == {want}
        seen.clear()


def test_calls_that_do_not_fit_are_refused(exact):
    m = _model()
    ids = torch.randint(2, 97, (2, 6), generator=torch.Generator().manual_seed(1))
    for kw in (dict(batch=0, max_len=8), dict(batch=1, max_len=0), dict(batch=1, max_len=8, sinks=-1)):
        with pytest.raises(ValueError):
            Mo.cobalt_cache(m, **kw)
    with pytest.raises(ValueError, match="pages of"):
        m(ids, past_key_values=Mo.cobalt_cache(m, 2, 8, page=24))
    with pytest.raises(ValueError, match="for 8 tokens"):
        m(torch.cat([ids, ids], 1), past_key_values=Mo.cobalt_cache(m, 2, 8))
    with pytest.raises(ValueError, match="for 3 sequences"):
        m(ids, past_key_values=Mo.cobalt_cache(m, 3, 8))
    with pytest.raises(ValueError, match="past_key_values"):
        m(ids)
    for bad in ([1, 1, 1, 1, 1, 0], [1, 0, 1, 1, 1, 1]):                # behind a sequence, inside it
        with pytest.raises(ValueError, match="in front"):
            m(ids, past_key_values=Mo.cobalt_cache(m, 2, 16), attention_mask=torch.tensor([[1] * 6, bad]))
    cache = Mo.cobalt_cache(m, 2, 16)
    m(ids, past_key_values=cache)
    with pytest.raises(ValueError, match="first call"):                 # padding that the first call did not have
        m(ids[:, :1], past_key_values=cache, attention_mask=torch.tensor([[0] + [1] * 6, [1] * 7]))
    with pytest.raises(NotImplementedError):
        m.generate(ids, past_key_values=Mo.cobalt_cache(m, 4, 32), num_beams=2, max_new_tokens=2, attention_mask=torch.ones_like(ids))
    m.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no_grad"):
        m(ids, past_key_values=Mo.cobalt_cache(m, 2, 16))
    m.requires_grad_(False)
    m.model.layers[0].self_attn.is_causal = False
    with pytest.raises(ValueError, match="causal"):
        m(ids, past_key_values=Mo.cobalt_cache(m, 2, 16))


def test_a_step_that_is_refused_leaves_the_lengths(exact):
    m = _model()
    cache = Mo.cobalt_cache(m, 1, 8)
    ids = torch.arange(2, 8)[None]
    m(ids, past_key_values=cache)
    with pytest.raises(ValueError):
        m(ids, past_key_values=cache)
    assert int(cache.get_seq_length()) == 6 and cache.layers[0].sequences.lens.tolist() == [6]


def test_windows_of_the_configuration_hold_where_a_model_passes_none(exact, monkeypatch):
    cfg = tr.Qwen2Config(vocab_size=97, hidden_size=128, intermediate_size=128, num_hidden_layers=3, num_attention_heads=2, num_key_value_heads=1,
                         use_sliding_window=True, sliding_window=6, max_window_layers=1)
    m = tr.Qwen2ForCausalLM(cfg).double().eval().requires_grad_(False)
    seen = []
    real = hf.cobalt_attention
    monkeypatch.setattr(hf, "cobalt_attention", lambda mod, q, k, v, mask, **kw: real(mod, q, k, v, mask, **{**kw, "sliding_window": None}))
    attend = hf.ops.cache_attention
    monkeypatch.setattr(hf.ops, "cache_attention", lambda *a, **k: seen.append(k["window"]) or attend(*a, **k))
    ids = torch.arange(2, 22)[None]
    want = m(ids).logits
    got = m(ids, past_key_values=Mo.cobalt_cache(m, 1, 32)).logits
    assert seen == [None, 6, 6] and float((got - want).abs().max()) < ATOL


def test_a_model_of_another_type_is_refused_before_the_lengths_advance():
    m = _model().float()
    cache = Mo.cobalt_cache(m, 1, 8)
    with pytest.raises(TypeError, match="float16"):
        m(torch.arange(2, 8)[None], past_key_values=cache)
    assert int(cache.get_seq_length()) == 0 and cache.layers[0].sequences.steps == 0


def _mixed(images="gemma3"):
    """Small decoders with a vision tower: Gemma 3, whose image tokens see one another, and Llava, which is causal throughout."""
    text = dict(vocab_size=97, hidden_size=128, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                head_dim=64, max_position_embeddings=512)
    vision = dict(hidden_size=32, intermediate_size=32, num_hidden_layers=2, num_attention_heads=2, image_size=28, patch_size=14)
    torch.manual_seed(3)
    if images == "gemma3":
        cfg = tr.Gemma3Config(text_config=tr.Gemma3TextConfig(**text, sliding_window=6, layer_types=["sliding_attention", "full_attention"]).to_dict(),
                              vision_config=tr.SiglipVisionConfig(**vision).to_dict(), mm_tokens_per_image=4, image_token_index=90,
                              boi_token_index=91, eoi_token_index=92)
        m = tr.Gemma3ForConditionalGeneration(cfg)
    else:
        cfg = tr.LlavaConfig(text_config=tr.MistralConfig(**text, sliding_window=None), vision_config=tr.CLIPVisionConfig(**vision), image_token_index=90)
        m = tr.LlavaForConditionalGeneration(cfg)
    return m.double().eval().requires_grad_(False)


def test_a_mask_that_says_more_than_causal_is_refused(exact):
    m = _mixed()
    ids = torch.arange(2, 22)[None]
    types = torch.zeros_like(ids)
    want = m(ids, token_type_ids=types).logits
    got = m(ids, token_type_ids=types, past_key_values=Mo.cobalt_cache(m, 1, 32)).logits
    assert float((got - want).abs().max()) < ATOL                       # text alone
    types[0, 4:8] = 1                                                   # an image: its tokens see one another
    cache = Mo.cobalt_cache(m, 1, 32)
    with pytest.raises(ValueError, match="causal"):
        m(ids, token_type_ids=types, past_key_values=cache)
    assert int(cache.get_seq_length()) == 0 and cache.layers[0].sequences.steps == 0


def test_masks_are_told_apart():
    mu = pytest.importorskip("transformers.masking_utils")
    causal, sliding = mu.causal_mask_function, mu.sliding_window_causal_mask_function
    mask = torch.ones(2, 9)
    hook = lambda f, size=None, n=9: hf._padding_mask(batch_size=2, q_length=n, kv_length=9, q_offset=9 - n, attention_mask=mask, mask_function=f, local_size=size)
    types = torch.tensor([[0, 0, 0, 0, 0, 0, 0, 0, 0], [0, 0, 1, 1, 0, 0, 0, 0, 0]])
    image = lambda b, h, q, k: (types[b, q] == 1) & (types[b, k] == 1)
    none = lambda b, h, q, k: (types[b, q] == 2) & (types[b, k] == 2)
    head = lambda b, h, q, k: (h == 0) & (q >= 0)
    for f, size in ((causal, None), (sliding(7), 7), (mu.or_masks(causal, none), None), (mu.or_masks(sliding(3), none), 3)):
        assert hook(f, size).data_ptr() == mask.data_ptr()
    assert hook(mu.or_masks(causal, image), None, 3).data_ptr() == mask.data_ptr()           # the image lies before the step's tokens
    for f, size in ((sliding(7), None), (sliding(6), 7), (causal, 7), (mu.or_masks(causal, image), None), (mu.or_masks(sliding(7), image), 7),
                    (mu.bidirectional_mask_function, None), (mu.and_masks(mu.packed_sequence_mask_function(types), causal), None), (mu.or_masks(causal, head), None)):
        with pytest.raises(ValueError, match="causal"):
            hook(f, size)


def test_masks_given_for_each_kind_of_layer_are_looked_at(exact):
    """A dictionary of masks reaches the layers as it is: none but the padding's own 2-D mask may be in it."""
    cfg = tr.Gemma3TextConfig(vocab_size=97, hidden_size=128, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
                              num_key_value_heads=2, head_dim=64, sliding_window=6, layer_types=["sliding_attention", "full_attention"])
    torch.manual_seed(3)
    m = tr.Gemma3ForCausalLM(cfg).double().eval().requires_grad_(False)
    ids = torch.arange(2, 12)[None]
    want = m(ids, attention_mask=torch.ones_like(ids)).logits
    real = torch.ones(1, 10)
    got = m(ids, attention_mask=dict(sliding_attention=real, full_attention=real.bool()), past_key_values=Mo.cobalt_cache(m, 1, 16)).logits
    assert float((got - want).abs().max()) < ATOL
    four, less = torch.zeros(1, 1, 10, 10), torch.ones(1, 7)
    for full in (four, less):
        with pytest.raises(ValueError, match="attention_mask must be"):
            m(ids, attention_mask=dict(sliding_attention=None, full_attention=full), past_key_values=Mo.cobalt_cache(m, 1, 16))
        with pytest.raises(ValueError, match="attention_mask must be"):
            m(ids, attention_mask=dict(sliding_attention=full, full_attention=None), past_key_values=Mo.cobalt_cache(m, 1, 16))
    pad = real.clone()
    pad[0, :3] = 0
    for masks in (dict(sliding_attention=real, full_attention=pad), dict(sliding_attention=None, full_attention=pad)):
        with pytest.raises(ValueError, match="the same padding"):
            m(ids, attention_mask=masks, past_key_values=Mo.cobalt_cache(m, 1, 16))
    cache = Mo.cobalt_cache(m, 1, 16)
    m(ids, attention_mask=dict(sliding_attention=pad, full_attention=pad.bool()), past_key_values=cache)
    m(ids[:, :1], attention_mask=dict(sliding_attention=torch.cat([pad, real[:, :1]], 1), full_attention=None), past_key_values=cache)
    assert cache.layers[0].sequences.lens.tolist() == [8]


def test_only_the_decoder_of_a_mixed_model_is_switched(exact):
    g = torch.Generator().manual_seed(2)
    m = _mixed("llava")
    ids = torch.randint(2, 90, (1, 12), generator=g)
    ids[0, 3:7] = 90                                                    # four patches of an image
    kw = dict(pixel_values=torch.randn(1, 3, 28, 28, dtype=torch.float64, generator=g))
    want = m(ids, **kw).logits
    dense = tr.DynamicCache(config=m.config.get_text_config())
    m(ids, past_key_values=dense, **kw)
    step = m(ids[:, :1], past_key_values=dense).logits
    cache = Mo.cobalt_cache(m, 1, 32)
    assert m.model.vision_tower.config._attn_implementation == "sdpa"
    assert float((m(ids, past_key_values=cache, **kw).logits - want).abs().max()) < ATOL
    assert float((m(ids[:, :1], past_key_values=cache).logits - step).abs().max()) < ATOL
    m.set_attn_implementation("sdpa")
    assert torch.equal(m(ids, **kw).logits, want)
    m = _mixed()                                                        # Gemma 3: its vision tower runs, its image is refused
    Mo.cobalt_cache(m, 1, 32)
    types = (ids == 90).long()
    with pytest.raises(ValueError, match="this step's mask"):
        m(ids, token_type_ids=types, past_key_values=Mo.cobalt_cache(m, 1, 32), **kw)


def test_an_eager_step_after_replays_goes_on_from_the_device(exact, monkeypatch):
    """A recorded step and its replays advance the lengths on the device, and no count on the host."""
    m = _model()
    ids = torch.randint(2, 97, (2, 17), generator=torch.Generator().manual_seed(4))
    mask = lambda n: torch.stack([(torch.arange(n) >= p).long() for p in (0, 3)])
    want = m(ids, attention_mask=mask(17)).logits
    recording = [False]
    monkeypatch.setattr(hf, "_recording", lambda: recording[0], raising=False)
    cache = Mo.cobalt_cache(m, 2, 18, page=16)
    seqs = cache.layers[0].sequences
    for _ in range(2):
        m(ids[:, :10], past_key_values=cache, attention_mask=mask(10))
        recording[0] = True
        for i in range(10, 14):                                         # what four replays do
            m(ids[:, i:i + 1], past_key_values=cache)
            seqs.steps = 10
        recording[0] = False
        got = m(ids[:, 14:17], past_key_values=cache, attention_mask=mask(17)).logits
        assert int(cache.get_seq_length()) == 17 and seqs.lens.tolist() == [17, 14]
        assert float((got - want[:, 14:]).abs().max()) < ATOL
        with pytest.raises(ValueError, match="for 18 tokens"):
            m(ids[:, :2], past_key_values=cache)
        recording[0] = True
        m(ids[:, :1], past_key_values=cache)                            # one more replay: no room is left
        recording[0] = False
        with pytest.raises(ValueError, match="for 18 tokens"):
            m(ids[:, :1], past_key_values=cache)
        cache.reset()                                                   # and anew: replays may follow a reset as well


def test_values_of_another_type_are_refused_before_the_lengths_advance(exact):
    m = _model()
    cache = Mo.cobalt_cache(m, 1, 16)
    ids = torch.arange(2, 8)[None]
    m(ids, past_key_values=cache)
    m.model.layers[0].self_attn.v_proj.register_forward_hook(lambda mod, args, out: out.float())
    with pytest.raises(TypeError, match="float16"):
        m(ids[:, :1], past_key_values=cache)
    assert int(cache.get_seq_length()) == 6 and cache.layers[0].sequences.lens.tolist() == [6]


def test_models_with_an_attention_of_their_own_are_refused(exact):
    """GPT-J's layers take no other attention function: they would attend over the step's own keys alone."""
    m = tr.GPTJForCausalLM(tr.GPTJConfig(vocab_size=97, n_embd=128, n_layer=2, n_head=2, rotary_dim=32)).double().eval().requires_grad_(False)
    with pytest.raises(ValueError, match="cannot be switched"):
        Mo.cobalt_cache(m, 1, 16)


def test_a_step_whose_layers_attend_otherwise_is_refused(exact):
    m = _model()
    ids = torch.arange(2, 8)[None]
    cache = Mo.cobalt_cache(m, 1, 32)
    m(ids, past_key_values=cache)
    m.set_attn_implementation("sdpa")                                   # switched back, and the cache passed on all the same
    with pytest.raises(RuntimeError, match="switched back"):
        m(ids[:, :1], past_key_values=cache)
    one = _model(layers=1)                                              # with a single layer the next call tells
    cache = Mo.cobalt_cache(one, 1, 32)
    one.set_attn_implementation("sdpa")
    one(ids, past_key_values=cache)
    with pytest.raises(RuntimeError, match="switched back"):
        one(ids, past_key_values=cache)
    cache.reset()
    one.set_attn_implementation("cobalt_cache")
    one(ids, past_key_values=cache)
    assert int(cache.get_seq_length()) == 6


@pytest.mark.parametrize("types,shared", [(["full_attention"] * 2, 1), (["sliding_attention", "full_attention"] * 2, 2)])
def test_layers_that_share_keys_and_values(exact, types, shared):
    """The last layers of Gemma 3n attend over what an earlier one has written, the very first among them."""
    cfg = tr.Gemma3nTextConfig(vocab_size=97, vocab_size_per_layer_input=97, hidden_size=128, intermediate_size=128, hidden_size_per_layer_input=32,
                               num_hidden_layers=len(types), num_attention_heads=2, num_key_value_heads=1, head_dim=64, max_position_embeddings=512,
                               sliding_window=6, layer_types=types, num_kv_shared_layers=shared, laurel_rank=8,
                               activation_sparsity_pattern=[0.0] * len(types), pad_token_id=0)
    torch.manual_seed(0)
    m = tr.Gemma3nForCausalLM(cfg).double().eval().requires_grad_(False)
    ids = torch.randint(2, 97, (2, 20), generator=torch.Generator().manual_seed(0))
    dense = tr.DynamicCache(config=m.config)
    want = [m(x, past_key_values=dense).logits for x in (ids[:, :15], ids[:, 15:16], ids[:, 16:])]
    cache = Mo.cobalt_cache(m, 2, 32)
    for i, x in enumerate((ids[:, :15], ids[:, 15:16], ids[:, 16:])):
        assert float((m(x, past_key_values=cache).logits - want[i]).abs().max()) < ATOL, i
    assert cache.layers[0].sequences.lens.tolist() == [20, 20]
