"""Steps of several tokens through the attention route and the batched store: which
masks they take, what precision their rows see and what can be taken back.

The host tests drive a small model or the store with the kernel calls recorded
instead of launched; the GPU tests compare whole steps."""

import pytest
import torch

from anchorkv_b200 import live


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
