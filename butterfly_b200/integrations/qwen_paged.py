"""Continuous batching for a Qwen3.5 model with its dense attention, over a paged cache.

The compressed path decodes a batch in lockstep from a two-pool cache.  The stock model that it
is compared with, or served beside, keeps every token: ``PagedQwenDecoder`` serves such a
model (full-attention layers, head_dim 128, not swapped) to requests of different lengths
that come and go.  A prompt runs through the model's own forward and its keys and values go
into pages (``paged_append``); a decode step advances all requests by one token:

    reserve (pages, lengths)                            once a step
    per layer:  rmsnorm + q/k/v projection, q/k norm + RoPE at each request's position,
                paged_decode_attention (writes the token's rows, attends), gate + o_proj +
                residual, rmsnorm + SwiGLU, down_proj + residual

with the fused glue of ``butterfly_b200.glue`` (weight-streaming GEMVs for up to 8 rows and input
sizes that are multiples of 256 up to 8,192).

    dec = PagedQwenDecoder(model, max_requests=8, num_pages=4096, max_tokens_per_request=32768)
    logits = dec.add({0: ids0, 3: ids3})                # {row: next-token logits}
    logits, granted = dec.step(tokens)                  # tokens [max_requests], rows not live ignored
    dec.finish([3])

``python -m butterfly_b200.integrations.qwen_paged`` runs a random-init model this way.
"""
from __future__ import annotations

from typing import Mapping, Sequence

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import glue
from ..paged import PagedKVCache, PagedReservation
from .qwen_fused import _is_qwen35_norm, _merge_weights
from .qwen_torch import _get_decoder_with_layers, _has_required_qwen_attention_attrs, patch_qwen35_full_attention_decode


class _Layer:
    def __init__(self, layer: nn.Module):
        attn, mlp = getattr(layer, "self_attn", None), getattr(layer, "mlp", None)
        if attn is None or mlp is None or not _has_required_qwen_attention_attrs(attn) or int(attn.head_dim) != 128:
            raise ValueError("PagedQwenDecoder needs dense Qwen3.5 full-attention layers with head_dim 128")
        norms = [getattr(attn, "q_norm", None), getattr(attn, "k_norm", None), layer.input_layernorm, layer.post_attention_layernorm]
        # (one launch normalises q and k, with one eps)
        if not all(_is_qwen35_norm(x) for x in norms) or norms[0].eps != norms[1].eps:
            raise ValueError("PagedQwenDecoder needs Qwen3.5 RMSNorms, q_norm and k_norm with one eps")
        if type(getattr(mlp, "act_fn", None)).__name__ not in ("SiLU", "SiLUActivation"):
            raise ValueError("PagedQwenDecoder needs the SiLU activation")
        if abs(float(getattr(attn, "scaling", 128 ** -0.5)) - 128 ** -0.5) > 1e-6:
            raise ValueError("PagedQwenDecoder needs attention scaled by head_dim ** -0.5")
        for lin in (attn.q_proj, attn.k_proj, attn.v_proj, attn.o_proj, mlp.gate_proj, mlp.up_proj, mlp.down_proj):
            if getattr(lin, "bias", None) is not None:
                raise ValueError("PagedQwenDecoder needs bias-free projections")
        self.attn, self.mlp, self.norm1, self.norm2 = attn, mlp, layer.input_layernorm, layer.post_attention_layernorm
        self.w_qkv = _merge_weights([attn.q_proj, attn.k_proj, attn.v_proj])
        self.w_gu = _merge_weights([mlp.gate_proj, mlp.up_proj])
        self.hq = attn.q_proj.out_features // 256  # a query and a gate row block per head
        self.hkv = attn.k_proj.out_features // 128
        self.inter = mlp.gate_proj.out_features


class PagedQwenDecoder:
    @torch.no_grad()
    def __init__(self, model: nn.Module, *, num_pages: int, max_tokens_per_request: int, max_requests: int = 8,
                 page_size: int = 64):
        patch_qwen35_full_attention_decode()
        self.model, self.decoder = model, _get_decoder_with_layers(model)
        head = getattr(model, "lm_head", None)
        if not _is_qwen35_norm(getattr(self.decoder, "norm", None)) or not isinstance(head, nn.Linear) or head.bias is not None:
            raise ValueError("PagedQwenDecoder needs a Qwen3.5 final norm and a bias-free lm_head")
        self.layers = [_Layer(layer) for layer in self.decoder.layers]
        w = self.layers[0].w_qkv
        self.cache = PagedKVCache(num_layers=len(self.layers), num_pages=num_pages, page_size=page_size,
                                  num_kv_heads=self.layers[0].hkv, head_dim=128, max_requests=max_requests,
                                  max_tokens_per_request=max_tokens_per_request, dtype=w.dtype, device=w.device)
        # the weight-streaming GEMVs take up to 8 rows, and inputs of these sizes; else library products
        sizes = [n for st in self.layers for n in (st.w_qkv.shape[1], 128 * st.hq, st.inter)]
        self._few = max_requests <= 8 and all(n % 256 == 0 and n <= 8192 for n in sizes)
        self.live = [False] * max_requests
        self._live_add = None  # device tensor of one token per live request, renewed when they change

    def _check_rows(self, rows: Sequence[int]) -> None:
        for b in rows:
            if not 0 <= b < self.cache.max_requests:
                raise ValueError(f"there is no row {b}: the cache has {self.cache.max_requests}")

    @torch.no_grad()
    def add(self, prompts: Mapping[int, torch.Tensor]) -> dict[int, torch.Tensor]:
        """Admit prompts (1-D token ids) into vacant rows; returns their next-token logits.  Raises
        RuntimeError if the pages do not suffice for all of them; nothing is admitted then, nor
        when the model's forward raises."""
        from transformers import DynamicCache
        rows = sorted(prompts)
        self._check_rows(rows)
        for b in rows:
            if self.live[b]:
                raise ValueError(f"row {b} is in use")
            if int(prompts[b].numel()) == 0:
                raise ValueError("a prompt needs at least one token")
        add = [int(prompts[b].numel()) if b in prompts else 0 for b in range(self.cache.max_requests)]
        r = self.cache.reserve(add)
        logits, at = {}, 0
        try:
            granted = r.granted.tolist()
            if not all(granted[b] for b in rows):
                raise RuntimeError("not enough free pages for the prompts")
            for b in rows:
                n = add[b]
                kv = DynamicCache(config=self.model.config)
                out = self.model(input_ids=prompts[b].reshape(1, n), past_key_values=kv, use_cache=True, logits_to_keep=1)
                for i, layer in enumerate(kv.layers):
                    self.cache.append(i, layer.keys[0].transpose(0, 1), layer.values[0].transpose(0, 1), r.slot_map[at:at + n])
                logits[b] = out.logits[0, -1]
                at += n
        except BaseException:  # the rows were vacant: nothing of them is kept
            self.cache.release(rows)
            raise
        for b in rows:
            self.live[b] = True
        self._live_add = None
        return logits

    def finish(self, rows: Sequence[int]) -> None:
        """Give the rows' pages back."""
        self._check_rows(rows)
        self.cache.release(rows)
        for b in rows:
            self.live[b] = False
        self._live_add = None

    @torch.no_grad()
    def step(self, tokens: torch.Tensor):
        """One token for every live request: ``tokens`` [max_requests] (entries of other rows do not
        matter, whatever they hold).  Returns the next-token logits [max_requests, vocab] and ``granted`` [max_requests]
        bool on the device: False for rows that are not live, or whose page could not be had
        (such a request stays as it was: finish others and step again).  If the step raises, all
        requests stay as they were."""
        R = self.cache.max_requests
        if self._live_add is None:
            self._live_add = torch.tensor([int(x) for x in self.live], dtype=torch.int32, device=self.cache.block_table.device)
        # rows that are not live embed token 0: their ids may be padding that no table holds
        ids = tokens.reshape(R, 1) * self._live_add[:, None]
        r = self.cache.reserve(self._live_add, sum(self.live))
        try:
            return self._forward(ids, r), r.granted
        except BaseException:  # a token without rows in every layer must not count
            self.cache.reserve(-(self._live_add * r.granted), 0)
            raise

    def _forward(self, ids: torch.Tensor, r: PagedReservation) -> torch.Tensor:
        R = self.cache.max_requests
        few = self._few
        pos = (r.lens - 1).clamp(min=0).long()[:, None]
        x = self.decoder.embed_tokens(ids)
        cos, sin = self.decoder.rotary_emb(x, pos)
        x = x.view(R, -1)
        for i, st in enumerate(self.layers):
            hq, hkv, a = st.hq, st.hkv, st.attn
            if few:
                qkv = glue.gemv_rmsnorm(x, st.norm1.weight, st.norm1.eps, st.w_qkv)
            else:
                qkv = F.linear(glue.rmsnorm(x, st.norm1.weight, st.norm1.eps), st.w_qkv)
            qg = qkv[:, :256 * hq].view(R, 1, hq, 256)  # per head: query, then gate
            k_raw = qkv[:, 256 * hq:256 * hq + 128 * hkv].view(R, 1, hkv, 128)
            v = qkv[:, 256 * hq + 128 * hkv:].view(R, 1, hkv, 128)
            q, k = glue.qk_norm_rope(qg[..., :128], k_raw, a.q_norm.weight, a.k_norm.weight, cos, sin, a.q_norm.eps)
            o = self.cache.attend(i, q.transpose(1, 2), k_new=k.transpose(1, 2), v_new=v.transpose(1, 2), active=r.granted)
            if few:
                x2 = glue.gemv_gated(o.view(R, hq, 128), qg[:, 0, :, 128:], a.o_proj.weight, residual=x)
                act = glue.gemv_rmsnorm(x2, st.norm2.weight, st.norm2.eps, st.w_gu, swiglu=True)
                x = glue.gemv(act, st.mlp.down_proj.weight, residual=x2)
            else:
                y = F.linear(glue.gate_sigmoid_mul(o.transpose(1, 2), qg[..., 128:]).view(R, 128 * hq), a.o_proj.weight)
                h, x2 = glue.rmsnorm(y, st.norm2.weight, st.norm2.eps, residual=x, want_sum=True)
                x = x2 + F.linear(glue.swiglu(F.linear(h, st.w_gu), st.inter), st.mlp.down_proj.weight)
        x = glue.rmsnorm(x, self.decoder.norm.weight, self.decoder.norm.eps)
        w = self.model.lm_head.weight
        return glue.gemv(x, w) if few else F.linear(x, w)


def main() -> None:
    import argparse
    import time

    from transformers import Qwen3_5TextConfig
    from transformers.models.qwen3_5.modeling_qwen3_5 import Qwen3_5ForCausalLM

    ap = argparse.ArgumentParser(description="continuous batching of a random-init Qwen3.5 model over a paged cache")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=4096, help="longest prompt; request i has a 1 / (i + 1) of it")
    ap.add_argument("--steps", type=int, default=64)
    args = ap.parse_args()
    if args.steps < 1:
        ap.error("--steps must be at least 1")
    untimed = min(3, args.steps - 1)
    cfg = Qwen3_5TextConfig(hidden_size=1024, num_attention_heads=8, num_key_value_heads=2, head_dim=128,
                            num_hidden_layers=args.layers, layer_types=["full_attention"] * args.layers,
                            intermediate_size=3584, vocab_size=32000, partial_rotary_factor=0.25)
    torch.manual_seed(0)
    model = Qwen3_5ForCausalLM(cfg).eval().to(torch.bfloat16).cuda()
    page = 64
    width = args.prompt + args.steps + page
    dec = PagedQwenDecoder(model, max_requests=args.requests, page_size=page, max_tokens_per_request=width,
                           num_pages=args.requests * -(-width // page))
    lens = [max(1, args.prompt // (i + 1)) for i in range(args.requests)]
    logits = dec.add({i: torch.randint(0, 32000, (n,), device="cuda") for i, n in enumerate(lens)})
    tokens = torch.stack([logits[i].argmax() for i in range(args.requests)])
    for s in range(args.steps):
        if s == untimed:
            torch.cuda.synchronize()
            t0 = time.perf_counter()
        logits, _ = dec.step(tokens)
        tokens = logits.argmax(-1)
    torch.cuda.synchronize()
    ms = (time.perf_counter() - t0) / (args.steps - untimed) * 1e3
    print(f"{args.requests} requests of {min(lens)} to {max(lens)} prompt tokens: {ms:.3f} ms a step, "
          f"{args.requests / ms * 1e3:.0f} tokens/s; lengths now {dec.cache.lens.tolist()}, "
          f"{int(dec.cache.num_free)} of {int(dec.cache.free_pages.numel())} pages free")


if __name__ == "__main__":
    main()

__all__ = ["PagedQwenDecoder"]
