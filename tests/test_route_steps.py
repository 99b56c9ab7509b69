"""Steps of several tokens through the attention route and the batched store: which
masks they take, what precision their rows see and what can be taken back.

The host tests drive a small model or the store with the kernel calls recorded
instead of launched; the GPU tests compare whole steps."""

import numpy as np
import pytest
import torch

import anchorkv_b200 as akv
from anchorkv_b200 import _lib, live
from anchorkv_b200 import pool as P


class _Reached(Exception):
    """The route got as far as the pages."""


class _NoPages:
    def batch_view(self, layer):
        raise _Reached

    def dense(self, layer):
        raise _Reached


def _tiny_model(**extra):
    from transformers import Qwen3Config, Qwen3ForCausalLM

    config = Qwen3Config(vocab_size=64, hidden_size=64, intermediate_size=64, num_hidden_layers=2,
                         num_attention_heads=2, num_key_value_heads=1, head_dim=32, attn_implementation="sdpa", **extra)
    return Qwen3ForCausalLM(config).eval()


def _cache_without_pages(held):
    from transformers import DynamicCache

    class Cache(DynamicCache):
        store = _NoPages()

        def get_seq_length(self, layer_idx=0):
            return held

        def update(self, key_states, value_states, layer_idx, cache_kwargs=None):
            return key_states, value_states

    return Cache()


@pytest.mark.parametrize("sliding", [None, 50])
@pytest.mark.parametrize("backend", ["packed", "dense"])
def test_masks_of_several_rows_are_refused(backend, sliding):
    """A padding mask or an explicit one changes what a row may see, which the pages' attention does not do."""
    extra = {} if sliding is None else dict(use_sliding_window=True, sliding_window=sliding, max_window_layers=0)
    model, held, rows = _tiny_model(**extra), 7, 3
    ids = torch.zeros((2, rows), dtype=torch.long)
    whole = torch.ones((2, held + rows), dtype=torch.long)
    left = whole.clone()
    left[1, :2] = 0
    tree = torch.ones((2, 1, rows, held + rows), dtype=torch.bool)
    cache = _cache_without_pages(held)

    def step(tokens, mask):
        with torch.no_grad(), live.paged_route(model, cache, backend):
            model(input_ids=tokens, past_key_values=cache, attention_mask=mask, use_cache=True)

    for mask in (left, tree, tree.float()):
        with pytest.raises(ValueError, match="several query tokens"):
            step(ids, mask)
    for mask in (None, whole):  # nothing hidden: the rows go on to the pages
        with pytest.raises(_Reached):
            step(ids, mask)
    for mask in (None, whole[:, :held + 1], left[:, :held + 1], tree[:, :, :1, :held + 1]):  # one token: as ever
        with pytest.raises(_Reached):
            step(ids[:, :1], mask)
    assert model.config._attn_implementation == "sdpa"


def test_the_mask_registry_is_restored():
    from transformers.masking_utils import ALL_MASK_ATTENTION_FUNCTIONS

    model, cache = _tiny_model(), _cache_without_pages(7)
    with live.paged_route(model, cache):
        assert ALL_MASK_ATTENTION_FUNCTIONS[live.ROUTE] is live._route_mask
    assert ALL_MASK_ATTENTION_FUNCTIONS[live.ROUTE] is ALL_MASK_ATTENTION_FUNCTIONS["sdpa"]


HEADS, DIM, LAYERS = 2, 64, 2


@pytest.fixture
def launches(monkeypatch):
    """Record C-ABI calls instead of launching them; keep descriptor arrays on the host."""
    calls = []
    monkeypatch.setattr(_lib, "call", lambda name, *args: calls.append(name))
    monkeypatch.setattr(_lib, "require_cuda", lambda *a, **k: None)
    monkeypatch.setattr(_lib, "raise_pending", lambda device: None)
    monkeypatch.setattr(_lib, "status_ptr", lambda device: 0)
    monkeypatch.setattr(_lib, "stream_of", lambda device: 0)
    monkeypatch.setattr(P, "to_device", lambda array, device: torch.from_numpy(np.ascontiguousarray(array, np.int64)))
    return calls


def _host_cache(prefix, batch=2, **kw):
    kv = torch.zeros((batch, HEADS, prefix, DIM), dtype=torch.float16)
    return live.batched_live_cache([(kv, kv)] * LAYERS, max_tokens=400, device="cpu", **kw)


def _step(cache, rows):
    kv = torch.zeros((cache.store.batch, HEADS, rows, DIM), dtype=torch.float16)
    for layer in range(LAYERS):
        cache.update(kv, kv, layer)


def _bits(store):
    assert (store.bits(0) == store.bits(1)).all() and (store.bits(0) == store.bits(0)[:1]).all()
    named = {b: int((store.bits(0) == b).sum()) * LAYERS for b in (4, 8, 16)}
    for b in (4, 8, 16):  # no page is shared here: every slot is free or named once
        assert store.pool.free_slots(b) + named[b] == store.pool.capacity[b]
    return store.bits(0)[0].tolist()


def test_a_step_of_several_tokens_keeps_its_pages_until_the_next(launches):
    """Pages that were recent before the step, and those that it writes, are FP16 while its rows attend them."""
    cache = _host_cache(70, recent_pages=2, protected=(1,))
    assert _bits(cache.store) == [4, 16, 16, 16, 16]              # complete: 4; recent: 2, 3
    _step(cache, 60)                                              # 130 tokens
    assert _bits(cache.store) == [4] + [16] * 8
    _step(cache, 3)                                               # 8 complete pages: 6 and 7 were recent
    assert _bits(cache.store) == [4, 16, 4, 4, 4, 4] + [16] * 3
    _step(cache, 1)
    assert _bits(cache.store) == [4, 16, 4, 4, 4, 4] + [16] * 3
    _step(cache, 200)                                             # 334 tokens
    _step(cache, 1)                                               # a single token demotes at once: 20 complete
    assert _bits(cache.store) == [4, 16] + [4] * 16 + [16] * 3
    assert cache.store.demotions == 2 * LAYERS * 17


@pytest.mark.parametrize("recent", [0, 1])
def test_rejected_drafts_are_cropped_across_page_borders(launches, recent):
    cache = _host_cache(30, recent_pages=recent)
    for keep in (31, 30, 33):
        _step(cache, 21 if recent else 5)  # completes the page that holds the accepted prefix, and more
        cache.crop(keep)
        assert cache.get_seq_length() == keep
        if keep > 30:
            cache.crop(30)
    assert _bits(cache.store) == [16 if recent else 4, 16]
    _step(cache, 3)
    _step(cache, 1)                        # accepted: 34 tokens
    assert _bits(cache.store) == ([4, 16, 16] if recent else [4, 4, 16])


def test_an_append_archives_at_once_unless_told(launches):
    cache = _host_cache(30, recent_pages=0)
    kv = torch.zeros((2, HEADS, 40, DIM), dtype=torch.float16)
    for layer in range(LAYERS):
        cache.store.append(layer, kv, kv)
    assert _bits(cache.store) == [4, 4, 4, 4, 16]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 37, 150])
@pytest.mark.parametrize("backend", ["packed", "dense"])
def test_a_steps_logits_do_not_see_its_own_archive(cuda, backend, rows):
    """A chunk over an INT4 store against the same chunk over a store whose pages from the recent window on
    are protected (always FP16): the same pages by value, so the same logits."""
    from transformers import DynamicCache, Qwen3Config, Qwen3ForCausalLM

    torch.manual_seed(5)
    config = Qwen3Config(vocab_size=256, hidden_size=256, intermediate_size=256, num_hidden_layers=2,
                         num_attention_heads=4, num_key_value_heads=2, head_dim=64, attn_implementation="sdpa")
    model = Qwen3ForCausalLM(config).to(device=cuda, dtype=torch.float16).eval()
    ids = torch.randint(0, 256, (2, 80 + rows), generator=torch.Generator().manual_seed(6)).to(cuda)
    logits = []
    with torch.inference_mode():
        stock = DynamicCache()
        model(input_ids=ids[:, :80], past_key_values=stock, use_cache=True, logits_to_keep=1)
        source = [(layer.keys, layer.values) for layer in stock.layers]
        for protected in ((), range(4, 20)):  # 5 complete pages, the last one recent
            cache = live.batched_live_cache(source, max_tokens=300, recent_pages=1, protected=protected, device=cuda)
            assert cache.store.bits(0)[0].tolist() == [4, 4, 4, 4, 16]
            with live.paged_route(model, cache, backend):
                logits.append(live.decode_step(model, cache, ids[:, 80:]))
    assert torch.equal(logits[0], logits[1])
    assert akv.take_device_status(cuda) == 0


@pytest.mark.parametrize("shape,rows", [((3,), 1), ((3, 1), 1), ((1, 3), 1), ((3, 2), 2), ((3, 3), 3)])
def test_a_token_per_sequence_comes_in_any_shape(launches, shape, rows):
    """As many tokens as sequences are one each, as before steps took several."""
    cache = _host_cache(20, batch=3)
    given = {}

    def model(input_ids, cache_position, logits_to_keep, **kw):
        given.update(ids=input_ids, at=cache_position, keep=logits_to_keep)
        return type("Out", (), {"logits": torch.zeros((*input_ids.shape, 5))})()

    tokens = torch.arange(3 * rows).view(shape)
    out = live.decode_step(model, cache, tokens)
    assert given["ids"].tolist() == tokens.reshape(3, rows).tolist()
    assert given["at"].tolist() == list(range(20, 20 + rows)) and given["keep"] == rows
    assert out.shape == ((3, 5) if rows == 1 else (3, rows, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,group,archive,recent,protected", [
    (128, 64, 4, 1, (1,)), (64, 32, 8, 2, ()), (128, 128, 16, 2, ()), (64, 64, 4, 0, (0, 5))])
def test_steps_with_forks_crops_and_compaction(cuda, dim, group, archive, recent, protected):
    """Pages that wait for the archive are shared, reopened, copied and moved like others; every step is
    checked against the token histories."""
    from test_gpu_store import LAYERS as STORE_LAYERS
    from test_gpu_store import _Histories

    class Steps(_Histories):
        def step(self, n):
            ids, before = self._new(n), len(self.tokens[0])
            for layer in range(STORE_LAYERS):
                self.store.append(layer, *self._kv(ids, layer), archive=False)
            self.tokens = [t + i.tolist() for t, i in zip(self.tokens, ids)]
            self.old = max(self.old, before // 16 - self.recent - 1)
            self.check()

    h = Steps(cuda, dim, group, archive, recent, protected)
    h.prefill(30)
    h.step(37)                     # 67 tokens: pages 1 to 3 wait
    h.attend(37)
    h.fork([0, 1, 0, 0])           # waiting pages are shared
    h.check()
    h.crop(50)                     # into one that three sequences share
    h.check()
    h.step(5)
    h.attend(5, window=20, sinks=3)
    h.fork([2, 2, 1])
    h.step(40)                     # shared pages archived once
    h.crop(58)                     # back to what the step before wrote
    h.check()
    h.store.compact()
    h.check()
    h.step(60)
    h.store.compact()              # with pages that wait
    h.check()
    h.attend(60, window=64)
    h.append(1)                    # a single token archives at once
    h.check()
    h.step(3)
    h.append(40)
    h.check()
    h.attend(3)
    h.crop(0)
    h.check()
    h.step(20)
    h.attend(20)
