"""A Hugging Face decoder on the key/value cache in 4 or 8 bits: `model.cobalt_cache` builds the cache that is passed as
`past_key_values`; the model's attention layers then call `cobalt_attention`, which writes their keys and values with
`ops.cache_write` and reads the cache with `ops.cache_attention`, prompts and single tokens alike."""
from __future__ import annotations

from functools import partial
from types import FunctionType
from typing import Optional

import torch
from transformers import AttentionInterface, AttentionMaskInterface
from transformers.cache_utils import Cache, CacheLayerMixin
from transformers.masking_utils import causal_mask_function, sliding_window_causal_mask_function

from . import ops
from .cache import KVCache, KVCache8, KVPages, KVRows

NAME = "cobalt_cache"
DTYPES = (torch.float16, torch.bfloat16)


def _recording() -> bool:
    return torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()


class _Sequences:
    """What the layers of one cache share: the pages, the lengths, and the rows of the step under way."""

    def __init__(self, batch: int, max_len: int, page: int, device, pages: Optional[int] = None):
        if batch < 1 or max_len < 1:
            raise ValueError(f"batch and max_len must be at least 1, got {batch} and {max_len}")
        self.batch, self.max_len, self.page = batch, max_len, page
        per = -(-max_len // page)
        self.pages = batch * per if pages is None else pages
        # each sequence has pages for all of `max_len`, or they take them as they grow
        self.tables = None if pages is None else KVPages(pages, batch, max_len, page=page, device=device)
        self.table = torch.arange(self.pages, dtype=torch.int32, device=device).view(batch, per) if pages is None else self.tables.table
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)         # real tokens, padding left out
        self.seen = torch.zeros((), dtype=torch.int64, device=device)            # tokens with the padding
        self.waiting = False     # a layer has handed on its keys and values, which its attention has not taken yet
        self.recorded = False    # a step has been: its replays advance the lengths on the device alone
        self.clear(first=True)

    def clear(self, first: bool = False):
        self.lens.zero_()
        if self.tables is not None and not first:
            ops.cache_pages(self.tables, self.lens)
        self.seen.zero_()
        self.waiting = False
        self.steps = 0           # `seen` as the host knows it (issued())
        self.pads = [0] * self.batch
        self.rows: Optional[KVRows] = None
        self.mask: Optional[torch.Tensor] = None     # of the step under way, as the first layer got it
        self.first = True                            # that step is the first

    def attended(self):
        """Refuses a model some of whose layers attend by themselves, over what `update` gives them: the step's own keys and values."""
        if self.waiting:
            self.waiting = False
            raise RuntimeError('a layer that uses the cache has not called the attention "cobalt_cache": the model does not take it, or its '
                               "attention was switched back while the cache is in use")

    def issued(self) -> int:
        """Tokens with the padding so far.  Once a step has been recorded an eager one reads them back, which waits for the device;
        while a step is recorded they are what they were before it."""
        if self.recorded and not _recording():
            self.steps = int(self.seen)
        return self.steps

    def begin(self, batch: int, tokens: int, mask: Optional[torch.Tensor]):
        """The rows of a step of `tokens` tokens a sequence, called by the first layer; advances the lengths."""
        if batch != self.batch:
            raise ValueError(f"the cache is for {self.batch} sequences, the step has {batch}")
        steps = self.issued()
        if steps + tokens > self.max_len:
            raise ValueError(f"the cache is for {self.max_len} tokens a sequence, the step ends at {steps + tokens}")
        first = steps == 0
        if mask is not None:
            self._shape(mask, steps + tokens)
            pads = self._pads(mask)
            if first:
                self.pads = pads
            elif pads != self.pads:
                raise ValueError("attention_mask: padding belongs in front of a sequence, in the first call")
        if self.tables is not None:
            need = sum(-(-(steps + tokens - p) // self.page) for p in self.pads)
            if need > self.pages:
                if first:
                    self.pads = [0] * self.batch
                raise ValueError(f"the cache has {self.pages} pages of {self.page} tokens, the step ends with {need}")
        self.mask, self.first = mask, first
        if _recording():
            self.recorded = True
        else:
            self.steps += tokens
        self.seen.add_(tokens)
        self.lens.add_(tokens)
        padded = first and any(self.pads)
        if padded:
            pads = torch.tensor(self.pads, dtype=torch.int32).to(self.lens.device)
            self.lens.sub_(pads)
        if self.tables is not None:                                 # (a replay that they do not last for: tokens without pages, not written)
            ops.cache_pages(self.tables, self.lens)
        self.rows = KVRows(self.table, self.lens)
        if padded:
            # the padding's rows belong to sequences of their own, which are empty and have no pages: not written, and 0 as the answer
            ends = torch.arange(batch, dtype=torch.int32, device=pads.device) * tokens
            starts = torch.stack([ends, ends + pads], 1).flatten()
            self.rows = KVRows(torch.stack([torch.full_like(self.table, -1), self.table], 1).flatten(0, 1).contiguous(),
                               torch.stack([torch.zeros_like(self.lens), self.lens], 1).flatten(),
                               torch.cat([starts, starts.new_full((1,), batch * tokens)]))

    def same_mask(self, mask: Optional[torch.Tensor]):
        """The mask of a further layer: a dictionary of masks by kinds of layers reaches them as it is, and all must say the same."""
        if mask is self.mask:
            return
        if mask is not None and (self.mask is None or mask.shape != self.mask.shape):
            self._shape(mask, self.issued())
        if getattr(mask, "_cobalt_hook", False) and getattr(self.mask, "_cobalt_hook", False):
            return                                                              # both of the one mask the model was called with
        pads = self._pads(mask) if mask is not None else [0] * self.batch if self.first else self.pads
        if pads != self.pads:
            raise ValueError("attention_mask: all layers must have the same padding")

    def _shape(self, mask, total):
        if mask.dim() != 2 or mask.shape[0] != self.batch or mask.shape[1] != total:
            raise ValueError(f"attention_mask must be [{self.batch}, {total}], got {list(mask.shape)}")

    def _pads(self, mask):
        if mask.is_cuda and _recording():
            raise ValueError("attention_mask is read by the host: a step recorded in a graph takes none (padding of the first call stays left out)")
        real = mask.bool()
        holes = (real[:, :-1] & ~real[:, 1:]).any(1)
        pads = torch.where(holes, -1, (~real).sum(1)).tolist()
        if -1 in pads:
            raise ValueError("attention_mask: padding belongs in front of a sequence, in the first call")
        return pads


class CobaltCacheLayer(CacheLayerMixin):
    """One decoder layer's pool.  `update` only hands the step's keys and values on: `cobalt_attention` writes them."""
    is_compileable = False
    is_sliding = False

    def __init__(self, sequences: _Sequences, index: int, make_pool, window: Optional[int], sinks: int):
        super().__init__()
        self.sequences, self.index, self.make_pool, self.window, self.sinks = sequences, index, make_pool, window, sinks
        self.pool = None

    def lazy_initialization(self, key_states, value_states):
        if key_states.shape != value_states.shape:
            raise ValueError(f"keys {list(key_states.shape)} and values {list(value_states.shape)} must have the same shape")
        if key_states.is_cuda and _recording():
            raise RuntimeError("the first call with a new cache makes its pages: it cannot be recorded in a graph")
        self.pool = self.make_pool(self.sequences.pages, key_states.shape[1], key_states.shape[3], page=self.sequences.page, device=key_states.device)
        self.is_initialized = True

    def update(self, key_states, value_states, *args, **kwargs):
        if self.pool is None:
            self.lazy_initialization(key_states, value_states)
        self.sequences.attended()
        self.sequences.waiting = True
        key_states._cobalt_layer = self
        return key_states, value_states

    def get_seq_length(self):
        return self.sequences.seen

    def get_mask_sizes(self, query_length):
        tokens = query_length if isinstance(query_length, int) else query_length.shape[0]
        return self.sequences.issued() + tokens, 0

    def get_max_cache_shape(self):
        return self.sequences.max_len

    get_max_length = get_max_cache_shape

    def reset(self):
        self.sequences.clear()

    def _refuse(self, *args, **kwargs):
        raise NotImplementedError("this cache does not reorder, repeat, select or crop its sequences, and is not offloaded")

    reorder_cache = batch_repeat_interleave = batch_select_indices = crop = offload = prefetch = _refuse


def cobalt_attention(module, query, key, value, attention_mask, scaling=None, dropout=0.0, sliding_window=None, **kwargs):
    """The attention function behind the name "cobalt_cache": query [batch, heads, tokens, head_dim] -> [batch, tokens, heads, head_dim]."""
    layer = getattr(key, "_cobalt_layer", None)
    if layer is None:
        raise ValueError('attention "cobalt_cache" needs a cache of model.cobalt_cache as past_key_values')
    fresh, layer.sequences.waiting = layer.sequences.waiting, False    # (not fresh: a layer that shares the keys and values of an earlier one)
    if dropout or kwargs.get("softcap") is not None or kwargs.get("s_aux") is not None or not getattr(module, "is_causal", True) \
            or kwargs.get("is_causal") is False:
        raise ValueError("attention over this cache is causal, without dropout, soft caps or learned sinks")
    if query.requires_grad or key.requires_grad or value.requires_grad:
        raise RuntimeError("this cache has no backward pass: call the model under torch.no_grad()")
    types = {x.dtype for x in (query, key, value)}
    if len(types) > 1 or not types <= set(DTYPES):                   # (before the lengths advance)
        raise TypeError(f"this cache is for float16 and bfloat16 models, not {', '.join(sorted(map(str, types)))}")
    batch, _, tokens, _ = query.shape
    window = sliding_window or layer.window                          # (models that leave it to their mask do not pass one)
    if layer.index == 0 and fresh:
        layer.sequences.begin(batch, tokens, attention_mask)
    else:
        layer.sequences.same_mask(attention_mask)
    as_rows = lambda x: x.transpose(1, 2).reshape(batch * tokens, x.shape[1], x.shape[3])
    if fresh:
        ops.cache_write(layer.pool, as_rows(key), as_rows(value), layer.sequences.rows)
    out = ops.cache_attention(layer.pool, as_rows(query), layer.sequences.rows, scale=scaling, window=window,
                              sinks=layer.sinks if window else 0)
    return out.view(batch, tokens, query.shape[1], query.shape[3]), None


def _same(a, b) -> bool:
    """Whether two mask functions are of the same code over the same values (the library builds new closures for every step)."""
    if isinstance(a, (tuple, list)) and isinstance(b, (tuple, list)):
        return len(a) == len(b) and all(map(_same, a, b))
    if isinstance(a, FunctionType) and isinstance(b, FunctionType):
        inner = lambda f: [c.cell_contents for c in f.__closure__ or ()]
        return a.__code__ is b.__code__ and _same(inner(a), inner(b))
    return type(a) is type(b) and isinstance(a, (int, float, str, type(None))) and a == b


def _answers_alike(f, plain, batch, heads, q_length, kv_length, q_offset, kv_offset, device) -> bool:
    """Whether a mask function hides and shows what the plain one does, over the rows and tokens of a step; read by the host."""
    at = lambda first, n, dim: (first + torch.arange(n, device=device)).view([n if d == dim else 1 for d in range(4)])
    b, h, kv = at(0, batch, 0), at(0, heads, 1), at(kv_offset, kv_length, 3)
    rows = max(1, (1 << 24) // (batch * kv_length))                     # at a time: 16 MB of truth values (a head)
    for i in range(0, q_length, rows):
        q = at(q_offset + i, min(rows, q_length - i), 2)
        if not bool((f(b, h, q, kv) == plain(b, h, q, kv)).all()):
            return False
    return True


def _padding_mask(batch_size=1, q_length=1, kv_length=1, q_offset=0, kv_offset=0, mask_function=causal_mask_function, attention_mask=None,
                  local_size=None, config=None, device=None, **kwargs):
    """The 2-D mask of the padding as it is.  What else the mask function says follows from the lengths and the window, if it is the
    plain causal or sliding one, or answers as that does (an image's tokens see one another, in a step without an image); any other is
    refused."""
    if local_size is not None:
        plain = [sliding_window_causal_mask_function(local_size)]
    else:                                                               # (with something added to it, the window is not told)
        size = getattr(config, "sliding_window", None)
        plain = [causal_mask_function] + ([sliding_window_causal_mask_function(size)] if size else [])
    mask = None
    if attention_mask is not None:
        mask = attention_mask.view(attention_mask.shape)                # one of its own, which the layers know to come from here
        mask._cobalt_hook = True
    if any(_same(mask_function, f) for f in plain):
        return mask
    if _recording():
        raise ValueError("a mask that a model adds to the causal one is read by the host: such a step cannot be recorded in a graph")
    heads = getattr(config, "num_attention_heads", 1)
    if not any(_answers_alike(mask_function, f, batch_size, heads, q_length, kv_length, q_offset, kv_offset, device) for f in plain):
        raise ValueError("attention over this cache is causal, under a sliding window at most: this step's mask says otherwise "
                         "(tokens that see later ones, or blocks that are kept apart)")
    return mask


def build(model, batch: int, max_len: int, page: int, group: int, sinks: int, bits: int = 4, block: int = 16, pages: Optional[int] = None) -> Cache:
    if bits not in (4, 8):
        raise ValueError(f"the cache holds 4 or 8 bits a value, not {bits}")
    make_pool = partial(KVCache, group=group) if bits == 4 else partial(KVCache8, block=block)
    cfg = model.config.get_text_config()
    types = getattr(cfg, "layer_types", None) or ["full_attention"] * cfg.num_hidden_layers
    kinds = set(types)
    if kinds - {"full_attention", "sliding_attention"} or getattr(model.config, "is_encoder_decoder", False):
        raise ValueError(f"this cache is for decoders of full and sliding-window attention, not {sorted(kinds)}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    AttentionInterface.register(NAME, cobalt_attention)
    AttentionMaskInterface.register(NAME, _padding_mask)
    seqs = _Sequences(batch, max_len, page, next(model.parameters()).device, pages)
    window = lambda kind: getattr(cfg, "sliding_window", None) if kind == "sliding_attention" else None
    cache = Cache(layers=[CobaltCacheLayer(seqs, i, make_pool, window(kind), sinks) for i, kind in enumerate(types)])
    decoder = model.get_decoder() or model                              # (a vision tower of the same model keeps its own)
    decoder.set_attn_implementation(NAME)
    if decoder.config._attn_implementation != NAME:
        raise ValueError(f"{type(decoder).__name__} has an attention of its own that cannot be switched: no such cache for it")
    return cache
