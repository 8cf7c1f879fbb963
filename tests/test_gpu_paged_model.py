"""A dense Qwen3.5 model served from a paged cache against its own forward, request by request.

The served logits of every step (tokens forced to the reference's) must stay within 3e-2 of the
stock model's, relative to the largest logit: the bar of the fused layers that the decode step
is made of (tests/test_gpu_glue.py)."""
import pytest
import torch

pytest.importorskip("transformers")
from transformers import DynamicCache, Qwen3_5TextConfig  # noqa: E402
from transformers.models.qwen3_5.modeling_qwen3_5 import Qwen3_5ForCausalLM  # noqa: E402

from butterfly_b200.integrations import qwen_torch as qt  # noqa: E402
from butterfly_b200.integrations.qwen_paged import PagedQwenDecoder  # noqa: E402

pytestmark = pytest.mark.gpu


def _model():
    qt.patch_qwen35_full_attention_decode()
    cfg = Qwen3_5TextConfig(hidden_size=512, num_attention_heads=8, num_key_value_heads=2, head_dim=128,
                            num_hidden_layers=3, layer_types=["full_attention"] * 3, intermediate_size=768,
                            vocab_size=1000, partial_rotary_factor=0.25)
    torch.manual_seed(1)
    return Qwen3_5ForCausalLM(cfg).eval().to(torch.bfloat16).cuda()


def _ids(n, seed):
    return torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(seed)).cuda()


class _Stock:
    @torch.no_grad()
    def __init__(self, model, ids):
        self.model, self.cache = model, DynamicCache(config=model.config)
        self.logits = model(input_ids=ids[None], past_key_values=self.cache, use_cache=True).logits[0, -1]

    @torch.no_grad()
    def step(self, token):
        self.logits = self.model(input_ids=token.view(1, 1), past_key_values=self.cache, use_cache=True).logits[0, -1]


def _close(a, b):
    assert float((a.float() - b.float()).abs().max()) <= 3e-2 * float(b.float().abs().max())


@pytest.mark.parametrize("rows", [4, 10])
def test_served_requests_match_the_stock_model(rows):
    model = _model()
    dec = PagedQwenDecoder(model, max_requests=rows, num_pages=24, page_size=16, max_tokens_per_request=256)
    prompts = {0: _ids(5, 1), 2: _ids(130, 2), 3: _ids(47, 3)}
    stock = {b: _Stock(model, x) for b, x in prompts.items()}
    for b, lg in dec.add(prompts).items():
        _close(lg, stock[b].logits)
    for s in range(6):
        if s == 3:  # one request leaves, another takes over its pages and a third row
            dec.finish([2])
            stock.pop(2)
            stock[1] = _Stock(model, _ids(100, 4))
            _close(dec.add({1: _ids(100, 4)})[1], stock[1].logits)
        tokens = torch.zeros(rows, dtype=torch.long, device="cuda")
        for b, ref in stock.items():
            tokens[b] = ref.logits.argmax()
        logits, granted = dec.step(tokens)
        assert [b for b, g in enumerate(granted.tolist()) if g] == sorted(stock)
        for b, ref in stock.items():
            ref.step(tokens[b])
            _close(logits[b], ref.logits)


def test_requests_without_room_wait():
    model = _model()
    dec = PagedQwenDecoder(model, max_requests=2, num_pages=3, page_size=16, max_tokens_per_request=64)
    with pytest.raises(RuntimeError, match="free pages"):
        dec.add({0: _ids(40, 1), 1: _ids(16, 2)})
    assert dec.cache.lens.tolist() == [0, 0] and int(dec.cache.num_free) == 3
    a, b = _Stock(model, _ids(16, 5)), _Stock(model, _ids(32, 6))
    dec.add({0: _ids(16, 5), 1: _ids(32, 6)})  # all three pages are full
    tokens = torch.stack([a.logits.argmax(), b.logits.argmax()])
    _, granted = dec.step(tokens)
    assert granted.tolist() == [False, False] and dec.cache.lens.tolist() == [16, 32]
    dec.finish([1])
    logits, granted = dec.step(tokens)
    assert granted.tolist() == [True, False]
    a.step(tokens[0])
    _close(logits[0], a.logits)


def test_refusals():
    model = _model()
    dec = PagedQwenDecoder(model, max_requests=2, num_pages=8, page_size=16, max_tokens_per_request=64)
    dec.add({0: _ids(3, 1)})
    with pytest.raises(ValueError, match="in use"):
        dec.add({0: _ids(3, 1)})
    with pytest.raises(ValueError, match="at least one token"):
        dec.add({1: _ids(0, 1)})
    qt.swap_qwen_attention_with_butterfly_cuda(model, qt.compressed_config())
    with pytest.raises(ValueError, match="dense"):
        PagedQwenDecoder(model, max_requests=2, num_pages=8, page_size=16, max_tokens_per_request=64)
