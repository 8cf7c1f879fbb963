"""Serving over the paged cache at model sizes that the weight-streaming projections take and do not take,
against the stock model; bars as in tests/test_gpu_paged_model.py."""
import pytest
import torch

pytest.importorskip("transformers")
from transformers import Qwen3_5TextConfig  # noqa: E402
from transformers.models.qwen3_5.modeling_qwen3_5 import Qwen3_5ForCausalLM  # noqa: E402

from butterfly_b200.integrations import qwen_torch as qt  # noqa: E402
from butterfly_b200.integrations.qwen_paged import PagedQwenDecoder  # noqa: E402

pytestmark = pytest.mark.gpu


def _model(inter=768, heads=8):
    qt.patch_qwen35_full_attention_decode()
    cfg = Qwen3_5TextConfig(hidden_size=512, num_attention_heads=heads, num_key_value_heads=2, head_dim=128,
                            num_hidden_layers=2, layer_types=["full_attention"] * 2, intermediate_size=inter,
                            vocab_size=1000, partial_rotary_factor=0.25)
    torch.manual_seed(1)
    return Qwen3_5ForCausalLM(cfg).eval().to(torch.bfloat16).cuda()


def _ids(n, seed):
    return torch.randint(0, 1000, (n,), generator=torch.Generator().manual_seed(seed)).cuda()


@torch.no_grad()
@pytest.mark.parametrize("inter,heads", [(640, 8), (8448, 8), (768, 16)])
@pytest.mark.parametrize("rows", [2, 8])
def test_intermediate_sizes(inter, heads, rows):
    model = _model(inter, heads)
    dec = PagedQwenDecoder(model, max_requests=rows, num_pages=24, page_size=16, max_tokens_per_request=128)
    prompts = {0: _ids(5, 1), rows - 1: _ids(37, 2)}
    logits = dec.add(prompts)
    for _ in range(2):
        tokens = torch.zeros(rows, dtype=torch.long, device="cuda")
        for b in prompts:
            tokens[b] = logits[b].argmax()
            prompts[b] = torch.cat([prompts[b], tokens[b:b + 1]])
        logits, granted = dec.step(tokens)
        assert granted.nonzero().flatten().tolist() == [0, rows - 1]
        for b, ids in prompts.items():
            ref = model(input_ids=ids[None]).logits[0, -1].float()
            assert float((logits[b].float() - ref).abs().max()) <= 3e-2 * float(ref.abs().max())


@pytest.mark.parametrize("steps", [1, 3, 5])
def test_example_of_a_few_steps(steps, monkeypatch, capsys):
    from butterfly_b200.integrations import qwen_paged
    monkeypatch.setattr("sys.argv", ["qwen_paged", "--layers", "1", "--requests", "2", "--prompt", "40", "--steps", str(steps)])
    qwen_paged.main()
    assert f"lengths now [{40 + steps}, {20 + steps}]" in capsys.readouterr().out
