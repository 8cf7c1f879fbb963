"""A dense Qwen3.5 model served from a 4-bit paged cache, the cache's calls one after another, and log probabilities of what it answers.

The reference is the stock model whose cache holds the rows that the pages hold (a code may be the next one where
the step's own rounding of a row lies beside a border, so that rows packed from the stock model's would not do).
Logits must stay within 3e-2 of its own, relative to the largest: the bar of the fused layers that
the decode step is made of (tests/test_gpu_glue.py)."""
import math

import pytest
import torch

pytest.importorskip("transformers")
from transformers import DynamicCache, Qwen3_5TextConfig  # noqa: E402
from transformers.models.qwen3_5.modeling_qwen3_5 import Qwen3_5ForCausalLM  # noqa: E402

import butterfly_b200 as bb  # noqa: E402
from butterfly_b200.integrations import qwen_torch as qt  # noqa: E402
from butterfly_b200.integrations.quality_smoke import prompt_scores  # noqa: E402
from butterfly_b200.integrations.qwen_paged import PagedQwenDecoder  # noqa: E402

from .test_gpu_paged_int4 import value  # noqa: E402

pytestmark = pytest.mark.gpu
VOCAB = 1000


def _model():
    qt.patch_qwen35_full_attention_decode()
    cfg = Qwen3_5TextConfig(hidden_size=512, num_attention_heads=8, num_key_value_heads=2, head_dim=128,
                            num_hidden_layers=3, layer_types=["full_attention"] * 3, intermediate_size=768,
                            vocab_size=VOCAB, partial_rotary_factor=0.25)
    torch.manual_seed(1)
    return Qwen3_5ForCausalLM(cfg).eval().to(torch.bfloat16).cuda()


def _ids(n, seed):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).cuda()


class _Stock:
    """The stock model; the rows of its cache are those that the served request's pages hold."""

    @torch.no_grad()
    def __init__(self, model, ids):
        self.model, self.cache = model, DynamicCache(config=model.config)
        self.logits = model(input_ids=ids[None], past_key_values=self.cache, use_cache=True).logits[0, -1]

    def take(self, paged, b, first):
        """The pages' rows of the tokens from `first` on, [1, Hkv, tokens, dh] of every layer."""
        pos = torch.arange(first, int(paged.lens[b]), device="cuda")
        slots = paged.block_table[b, pos // paged.page_size].long() * paged.page_size + pos % paged.page_size
        return [[x.transpose(0, 1)[None] for x in paged.read(i, slots)] for i in range(len(self.cache.layers))]

    def admitted(self, paged, b):
        for layer, (k, v) in zip(self.cache.layers, self.take(paged, b, 0)):
            assert k.shape == layer.keys.shape
            # what was appended, held in 4 bits: the cached rows of this forward are those of the serving one
            assert torch.equal(k, value(layer.keys).to(k.dtype)) and torch.equal(v, value(layer.values).to(v.dtype))
            layer.keys, layer.values = k, v

    @torch.no_grad()
    def step(self, token, paged, b):
        new = self.take(paged, b, int(paged.lens[b]) - 1)
        updates = []
        for layer, (k, v) in zip(self.cache.layers, new):
            updates.append(layer.update)
            layer.update = lambda k0, v0, *a, k=k, v=v, plain=layer.update, **kw: plain(k, v, *a, **kw)
        self.logits = self.model(input_ids=token.view(1, 1), past_key_values=self.cache, use_cache=True).logits[0, -1]
        for layer, u in zip(self.cache.layers, updates):
            layer.update = u


def _close(a, b):
    assert float((a.float() - b.float()).abs().max()) <= 3e-2 * float(b.float().abs().max())


@pytest.mark.parametrize("rows", [4, 10])
def test_served_requests_match_the_stock_model_over_4_bits(rows):
    model = _model()
    dec = PagedQwenDecoder(model, max_requests=rows, num_pages=24, page_size=16, max_tokens_per_request=256, cache_bits=4)
    assert dec.cache.cache_bits == 4
    prompts = {0: _ids(5, 1), 2: _ids(130, 2), 3: _ids(47, 3)}
    stock = {b: _Stock(model, x) for b, x in prompts.items()}
    for b, lg in dec.add(prompts).items():
        _close(lg, stock[b].logits)
        stock[b].admitted(dec.cache, b)
    for s in range(6):
        if s == 3:  # one request leaves, another takes over its pages and a third row
            dec.finish([2])
            stock.pop(2)
            stock[1] = _Stock(model, _ids(100, 4))
            _close(dec.add({1: _ids(100, 4)})[1], stock[1].logits)
            stock[1].admitted(dec.cache, 1)
        tokens = torch.zeros(rows, dtype=torch.long, device="cuda")
        for b, st in stock.items():
            tokens[b] = st.logits.argmax()
        logits, granted = dec.step(tokens)
        r = bb.token_logprobs(logits, tokens, top_k=5)
        want = torch.log_softmax(logits.double(), -1)
        assert ((r.logprobs - want.gather(1, tokens[:, None])[:, 0]).abs() <= 1e-5).all()
        assert torch.equal(r.top_ids[:, 0], logits.float().argmax(-1))
        for b, st in stock.items():
            assert bool(granted[b])
            st.step(tokens[b], dec.cache, b)
            _close(logits[b], st.logits)


def test_a_captured_step_of_the_cache():
    """reserve, attend and read of a PagedKVCache in one graph: replays advance the requests, each equal to the eager step."""
    g = torch.Generator(device="cuda").manual_seed(0)
    B, Hq, Hkv, dh, page = 3, 8, 2, 128, 16

    def build():
        c = bb.PagedKVCache(num_layers=1, num_pages=40, page_size=page, num_kv_heads=Hkv, head_dim=dh, max_requests=B,
                            max_tokens_per_request=128, cache_bits=4)
        rows = torch.randn(50, Hkv, dh, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
        c.append(0, rows, -rows, c.reserve([7, 30, 13]).slot_map)
        return c

    q, kn, vn = (torch.randn(B, h, 1, dh, generator=g, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv))
    one = torch.ones(B, dtype=torch.int32, device="cuda")

    def step(c):
        r = c.reserve(one, B)
        out, lse = c.attend(0, q, k_new=kn, v_new=vn, active=r.granted, return_lse=True)
        return (out, lse, *c.read(0, r.slot_map))

    a, b = build(), build()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(a)
    for _ in range(20):
        graph.replay()
        want = step(b)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(captured, want))
    assert a.lens.tolist() == [27, 50, 33] and torch.equal(a.block_table, b.block_table)
    assert torch.equal(captured[2], value(kn[:, :, 0]).bfloat16()) and torch.equal(captured[3], value(vn[:, :, 0]).bfloat16())


def test_prompt_scores():
    model = _model()
    ids = _ids(333, 7)[None]
    with torch.no_grad():
        logp = torch.log_softmax(model(input_ids=ids).logits[0, :-1].double(), -1)
    nll = -float(logp.gather(1, ids[0, 1:, None]).mean())
    entropy = -float((logp.exp() * logp).sum(-1).mean())
    for chunk in (64, 1000):  # (library products of other row counts: bf16 logits off by a rounding, 2^-8 of at most ~4)
        s = prompt_scores(model, ids, chunk)
        assert abs(s["nll"] - nll) <= 2e-2 and abs(s["entropy"] - entropy) <= 2e-2
    assert math.isfinite(prompt_scores(model, ids[:, :1])["nll"])
