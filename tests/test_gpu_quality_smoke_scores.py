"""The prompt's scores of the quality smoke: asked for, for any model that answers a call, and those of the swapped model.

The bar of means over a prompt: logits from library products of other row counts may fall on the next bf16 value, 2^-8 of
at most about 4 each."""
import math

import pytest
import torch

pytest.importorskip("transformers")
from transformers import Qwen3_5TextConfig  # noqa: E402
from transformers.models.qwen3_5.modeling_qwen3_5 import Qwen3_5ForCausalLM  # noqa: E402

from butterfly_b200.integrations import qwen_torch as qt  # noqa: E402
from butterfly_b200.integrations.quality_smoke import prompt_ids, prompt_scores, quality_smoke  # noqa: E402
from butterfly_b200.integrations.qwen_fused import fuse_qwen_decoder_layers, unfuse_qwen_decoder_layers  # noqa: E402

pytestmark = pytest.mark.gpu
BAR = 2e-2


def _model():
    qt.patch_qwen35_full_attention_decode()
    cfg = Qwen3_5TextConfig(hidden_size=512, num_attention_heads=8, num_key_value_heads=2, head_dim=128, num_hidden_layers=2,
                            layer_types=["full_attention"] * 2, intermediate_size=1024, vocab_size=1000)
    torch.manual_seed(5)
    return Qwen3_5ForCausalLM(cfg).eval().to(torch.bfloat16).cuda()


@torch.no_grad()
def _scores(model, ids):
    logp = torch.log_softmax(model(input_ids=ids, use_cache=False).logits[0, :-1].double(), -1)
    return -float(logp.gather(1, ids[0, 1:, None]).mean()), -float((logp.exp() * logp).sum(-1).mean())


class _Call(torch.nn.Module):
    """A model with nothing to reach but its call."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, **kw):
        return self.inner(**kw)


def test_a_model_that_only_answers_calls():
    model, ids = _model(), prompt_ids(1000, 300).cuda()
    nll, entropy = _scores(model, ids)
    for m in (model, _Call(model)):
        s = prompt_scores(m, ids, 128)
        assert abs(s["nll"] - nll) <= BAR and abs(s["entropy"] - entropy) <= BAR


def test_scores_are_asked_for():
    model, ids = _model(), prompt_ids(1000, 4096).cuda()
    tokens = [0]
    handle = model.model.register_forward_hook(lambda m, a, kw, out: tokens.__setitem__(0, tokens[0] + kw["input_ids"].shape[1]),
                                               with_kwargs=True)
    plain = quality_smoke(model, ids, decode_len=2, top_k=20)
    assert not [k for k in plain["metrics"] if k.startswith("prompt_")]
    assert tokens[0] == 2 * (4096 + 1)  # each mode: the prompt and one token
    handle.remove()
    met = quality_smoke(model, ids, decode_len=2, top_k=20, score_prompt=True)["metrics"]
    want = {"stock": _scores(model, ids)}
    qt.swap_qwen_attention_with_butterfly_cuda(model, qt.compressed_config())
    fuse_qwen_decoder_layers(model)
    want["compressed"] = _scores(model, ids)
    unfuse_qwen_decoder_layers(model)
    qt.restore_qwen_dense_attention(model)
    assert want["stock"] != want["compressed"]
    for mode, (nll, entropy) in want.items():
        assert math.isfinite(nll) and abs(met[f"prompt_nll_{mode}"] - nll) <= BAR
        assert math.isfinite(entropy) and abs(met[f"prompt_entropy_{mode}"] - entropy) <= BAR
