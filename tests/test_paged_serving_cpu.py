"""Host logic of PagedQwenDecoder on the CPU: a stand-in cache keeps the lengths and free pages, the
kernels are replaced by plain functions, so that ids, failures and refusals can be followed
without a GPU."""
import pytest
import torch

pytest.importorskip("transformers")
from transformers import Qwen3_5TextConfig  # noqa: E402
from transformers.models.qwen3_5.modeling_qwen3_5 import Qwen3_5ForCausalLM  # noqa: E402

from butterfly_b200 import glue  # noqa: E402
from butterfly_b200.integrations import qwen_torch as qt  # noqa: E402
from butterfly_b200.integrations.qwen_paged import PagedQwenDecoder  # noqa: E402
from butterfly_b200.paged import RELEASE, PagedReservation  # noqa: E402

PAGE, ROWS, VOCAB = 16, 4, 500


def _model(layers=2):
    qt.patch_qwen35_full_attention_decode()
    cfg = Qwen3_5TextConfig(hidden_size=256, num_attention_heads=4, num_key_value_heads=1, head_dim=128,
                            num_hidden_layers=layers, layer_types=["full_attention"] * layers,
                            intermediate_size=256, vocab_size=VOCAB, partial_rotary_factor=0.25)
    torch.manual_seed(0)
    return Qwen3_5ForCausalLM(cfg).eval()


class _Cache:
    """Lengths, free pages and the appended slots of a PagedKVCache, on the host."""

    def __init__(self, pages=12):
        self.max_requests, self.lens, self.free = ROWS, torch.zeros(ROWS, dtype=torch.int32), pages
        self.block_table = torch.zeros(ROWS, 4, dtype=torch.int32)
        self.written = 0

    def reserve(self, add, num_tokens=None):
        add = [int(x) for x in add]
        assert num_tokens is None or num_tokens >= sum(max(x, 0) for x in add)
        granted, lens = [], self.lens.tolist()
        for b, a in enumerate(add):
            want = max(0, lens[b] + a)
            need = -(-want // PAGE) + (-lens[b] // PAGE)
            ok = need <= self.free
            granted.append(ok and a > 0)
            if ok:
                lens[b], self.free = want, self.free - need
        self.lens = torch.tensor(lens, dtype=torch.int32)
        total = sum(max(x, 0) for x in add)
        return PagedReservation(self.lens, torch.tensor([self.free]), torch.arange(total), torch.arange(total, dtype=torch.int32),
                                torch.tensor(granted))

    def release(self, rows):
        self.reserve([RELEASE if b in set(rows) else 0 for b in range(ROWS)])

    def append(self, layer, k, v, slots):
        assert k.shape[0] == v.shape[0] == slots.shape[0]
        self.written += 1

    def attend(self, layer, q, **kw):
        return torch.zeros(ROWS, q.shape[1], 1, 128, dtype=q.dtype)


@pytest.fixture
def dec(monkeypatch):
    """A decoder of no layers (what surrounds them is left) whose norm and head run on the CPU."""
    d = PagedQwenDecoder(_model(), max_requests=ROWS, num_pages=12, page_size=PAGE, max_tokens_per_request=64)
    d.cache, d.layers = _Cache(), []
    monkeypatch.setattr(glue, "rmsnorm", lambda x, w, eps, **kw: x)
    monkeypatch.setattr(glue, "gemv", lambda x, w, **kw: x @ w.t())
    return d


def _ids(n, seed=0):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed))


def test_ids_of_rows_that_are_not_live_do_not_matter(dec):
    dec.add({1: _ids(5)})
    tokens = torch.tensor([-1, 7, VOCAB, 2 ** 40])  # padding ids that no embedding table holds
    logits, granted = dec.step(tokens)
    assert granted.tolist() == [False, True, False, False]
    want = dec.model.lm_head(dec.decoder.embed_tokens(torch.tensor(7)))
    torch.testing.assert_close(logits[1], want)


def _state(d):
    return d.cache.lens.tolist(), d.cache.free, list(d.live)


@pytest.mark.parametrize("calls", [0, 1, 2])
def test_prompts_are_given_back_when_the_model_raises(dec, calls):
    dec.add({2: _ids(20)})
    before, forward, made = _state(dec), dec.model.forward, []

    def failing(*a, **kw):
        if len(made) == calls:
            raise MemoryError("out of memory")
        made.append(1)
        return forward(*a, **kw)

    dec.model.forward = failing
    prompts = {0: _ids(40, 1), 1: _ids(3, 2), 3: _ids(17, 3)}
    with pytest.raises(MemoryError):
        dec.add(prompts)
    assert _state(dec) == before
    assert dec.step(torch.zeros(ROWS, dtype=torch.long))[1].tolist() == [False, False, True, False]
    dec.model.forward = forward
    logits = dec.add(prompts)
    assert sorted(logits) == [0, 1, 3] and dec.live == [True] * 4 and dec.cache.lens.tolist() == [40, 3, 21, 17]


def test_prompts_are_given_back_when_an_append_raises(dec):
    before = _state(dec)
    dec.cache.append = lambda *a: (_ for _ in ()).throw(RuntimeError("append"))
    with pytest.raises(RuntimeError, match="append"):
        dec.add({0: _ids(40, 1), 1: _ids(3, 2)})
    assert _state(dec) == before


def test_a_step_that_raises_advances_no_request(dec, monkeypatch):
    dec.add({0: _ids(16, 1), 2: _ids(20, 2), 3: _ids(64, 3)})  # row 0 needs a page for its next token
    dec.cache.free = 1
    before = _state(dec)
    tokens = torch.zeros(ROWS, dtype=torch.long)
    with monkeypatch.context() as m:
        m.setattr(glue, "gemv", lambda *a, **kw: (_ for _ in ()).throw(RuntimeError("head")))
        for _ in range(2):
            with pytest.raises(RuntimeError, match="head"):
                dec.step(tokens)
            assert _state(dec) == before
    granted = dec.step(tokens)[1].tolist()
    assert granted == [True, False, True, False] and dec.cache.lens.tolist() == [17, 0, 21, 64]


@pytest.mark.parametrize("row", [-1, ROWS, ROWS + 3])
def test_rows_that_are_not_there(dec, row):
    dec.add({0: _ids(5), ROWS - 1: _ids(20)})
    before = _state(dec)
    with pytest.raises(ValueError, match="row"):
        dec.add({row: _ids(4), 1: _ids(3)})
    with pytest.raises(ValueError, match="row"):
        dec.finish([0, row])
    assert _state(dec) == before


def _plain_norm(n):
    return torch.nn.RMSNorm(n)


@pytest.mark.parametrize("change", [
    lambda m: setattr(m.model.layers[1].self_attn, "q_norm", _plain_norm(128)),
    lambda m: setattr(m.model.layers[1].self_attn, "k_norm", _plain_norm(128)),
    lambda m: setattr(m.model.layers[0], "input_layernorm", _plain_norm(256)),
    lambda m: setattr(m.model.layers[0], "post_attention_layernorm", _plain_norm(256)),
    lambda m: setattr(m.model.layers[0].self_attn.k_norm, "eps", 1e-3),
    lambda m: setattr(m.model.layers[0].self_attn, "scaling", 0.5),
    lambda m: setattr(m.model.layers[1].mlp, "act_fn", torch.nn.GELU()),
    lambda m: setattr(m.model, "norm", _plain_norm(256)),
    lambda m: setattr(m, "lm_head", torch.nn.Linear(256, VOCAB, bias=True)),
    lambda m: setattr(m.model.layers[1].mlp, "down_proj", torch.nn.Linear(256, 256, bias=True)),
])
def test_models_that_the_step_would_not_follow_are_refused(change):
    m = _model()
    change(m)
    with pytest.raises(ValueError, match="PagedQwenDecoder needs"):
        PagedQwenDecoder(m, max_requests=ROWS, num_pages=12, page_size=PAGE, max_tokens_per_request=64)
