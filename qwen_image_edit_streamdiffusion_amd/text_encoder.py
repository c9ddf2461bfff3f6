"""The prompt encoder's language model on the HIP path.

The reference encodes each prompt (and its condition image) with the pipeline's ``text_encoder``,
Qwen2.5-VL-7B [U: diffusers QwenImageEditPlusPipeline.encode_prompt -> transformers
Qwen2_5_VLForConditionalGeneration, hidden_states[-1]], invoked through server.py:137-153 and
qwen_realtime.py:140-165 (the prompt cache).  This module is its decoder-only language model
(``Qwen2_5_VLTextModel``): embed_tokens, N x (RMSNorm, q|k|v with bias, multimodal rotate-half
RoPE on 3-D positions, causal GQA attention, o_proj + residual, RMSNorm, SwiGLU MLP + residual),
final RMSNorm -- the hidden states the DiT consumes as ``encoder_hidden_states``.  The vision tower
that turns the condition image into the ``<|image_pad|>`` embeddings is the next half of f2;
``forward`` already takes those embeddings (``inputs_embeds`` rows) and their 3-D positions.

MI355X mapping: every projection is one GEMM (q|k|v packed, gate|up packed; o_proj and down_proj
carry the residual add in their epilogue), RMSNorm / RoPE / SwiGLU / embedding are HIP kernels,
attention runs all heads per launch: head-batched fp32 score GEMM (GQA: the kv operand advances once
per group), one causal softmax over every head's rows, head-batched P.V against V^T (prompt
lengths are a few hundred tokens, so the full score blocks stay small).

``forward_packed`` takes several prompts in one pass without padding (ops.rope_axes,
ops.attention_packed: no scores in memory), ``extend`` new tokens after what a PagedKVCache holds of
their sequences (ops.rope_append, ops.attention_paged). Their rotation has one rounding, fp32 angles
and tables none; ``packed_attention`` makes ``forward`` go the same way.
"""
from __future__ import annotations

import hashlib
import math
from collections import OrderedDict
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import ops
from .kv_cache import PagedKVCache
from .rope import section_turns

BF16 = torch.bfloat16


@dataclass
class TextEncoderConfig:
    """Qwen2_5_VLTextConfig fields the forward uses (defaults: Qwen2.5-VL-7B)."""

    vocab_size: int = 152064
    hidden_size: int = 3584
    intermediate_size: int = 18944
    num_hidden_layers: int = 28
    num_attention_heads: int = 28
    num_key_value_heads: int = 4
    rms_norm_eps: float = 1e-6
    rope_theta: float = 1000000.0
    mrope_section: Tuple[int, ...] = (16, 24, 24)

    @property
    def head_dim(self) -> int:
        return self.hidden_size // self.num_attention_heads


def mrope_tables(cfg: TextEncoderConfig, position_ids: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos / sin [S, head_dim] for 3-D positions [3, S] (temporal, height, width), as
    Qwen2_5_VLRotaryEmbedding + apply_multimodal_rotary_pos_emb build them: fp32 freqs =
    pos * inv_freq, emb = cat(freqs, freqs), cos / sin in fp32, section i of the doubled
    mrope_section taken from axis i % 3, cast to bf16."""
    Dh = cfg.head_dim
    inv = 1.0 / (cfg.rope_theta ** (torch.arange(0, Dh, 2, dtype=torch.float) / Dh))
    pos = position_ids.to(torch.float32).cpu()                       # [3, S]
    freqs = pos[:, :, None] * inv[None, None, :]                     # [3, S, Dh/2]
    emb = torch.cat([freqs, freqs], dim=-1)                          # [3, S, Dh]
    cos, sin = emb.cos(), emb.sin()
    sec = list(cfg.mrope_section) * 2
    parts_c, parts_s, o = [], [], 0
    for i, n in enumerate(sec):
        parts_c.append(cos[i % 3, :, o:o + n])
        parts_s.append(sin[i % 3, :, o:o + n])
        o += n
    return torch.cat(parts_c, -1).to(BF16), torch.cat(parts_s, -1).to(BF16)


def text_state_dict_shapes(c: TextEncoderConfig) -> Dict[str, Tuple[int, ...]]:
    """Qwen2_5_VLTextModel parameter names (text-model relative) and shapes."""
    D, F, Dh = c.hidden_size, c.intermediate_size, c.head_dim
    kv = c.num_key_value_heads * Dh
    out = {"embed_tokens.weight": (c.vocab_size, D), "norm.weight": (D,)}
    for i in range(c.num_hidden_layers):
        p = f"layers.{i}."
        out.update({p + "input_layernorm.weight": (D,), p + "post_attention_layernorm.weight": (D,),
                    p + "self_attn.q_proj.weight": (D, D), p + "self_attn.q_proj.bias": (D,),
                    p + "self_attn.k_proj.weight": (kv, D), p + "self_attn.k_proj.bias": (kv,),
                    p + "self_attn.v_proj.weight": (kv, D), p + "self_attn.v_proj.bias": (kv,),
                    p + "self_attn.o_proj.weight": (D, D), p + "mlp.gate_proj.weight": (F, D),
                    p + "mlp.up_proj.weight": (F, D), p + "mlp.down_proj.weight": (D, F)})
    return out


def random_state_dict(shapes: Dict[str, Tuple[int, ...]], device, seed: int = 0) -> Dict[str, torch.Tensor]:
    """Random-init bf16 weights generated on ``device`` (the checkpoint is not available offline):
    norms ~1, biases ~0.02, matrices ~N(0, 1/fan_in)."""
    g = torch.Generator(device=device).manual_seed(seed)
    sd = {}
    for k, s in shapes.items():
        if k.endswith("norm.weight") or "norm" in k.split(".")[-2] or "ln_q" in k:
            t = torch.ones(s, device=device)
        elif k.endswith("bias"):
            t = 0.02 * torch.randn(s, generator=g, device=device)
        else:
            t = torch.randn(s, generator=g, device=device) / math.sqrt(math.prod(s[1:]))
        sd[k] = t.to(BF16)
    return sd


def encoder_splits(M: int, N: int, K: int) -> int:
    """K ranges for an encoder linear: prompts are a few hundred rows, so a projection with a
    narrow N (o_proj, down_proj, the vision proj / down) fills only a fraction of the 256 CUs
    with 256x256 tiles; split K until tiles x splits reaches about one round, >= 8 K tiles each."""
    tiles = -(-M // 256) * -(-N // 256)
    steps = K * 2 // 128
    for sp in range(min(256 // tiles, steps // 8), 1, -1):
        if steps % sp == 0:
            return sp
    return 1


class EncoderLinears:
    """The encoders' projections: split-K (fp32 partials in a shared workspace, reduced in range
    order with the real epilogue) where encoder_splits says the unsplit grid is too small, the
    plain GEMM otherwise."""

    def __init__(self, device):
        self.device = device
        self.ws = torch.empty(0, dtype=torch.float32, device=device)

    def _workspace(self, M, N, sp):
        need = ops.splitk_workspace_bytes(M, N, sp) // 4
        if self.ws.numel() < need:
            self.ws = torch.empty(need, dtype=torch.float32, device=self.device)
        return self.ws

    def linear(self, x, w, b, out):
        M, K = x.shape
        sp = encoder_splits(M, w.shape[0], K)
        if sp == 1:
            return ops.linear(x, w, b, out=out)
        return ops.linear_splitk(x, w, b, ops.EPI_BIAS, out, self._workspace(M, w.shape[0], sp), sp)

    def residual(self, x, w, b, ones, resid):
        """resid += x.w^T + b (the gated-residual epilogue with a unit gate)."""
        M, K = x.shape
        sp = encoder_splits(M, w.shape[0], K)
        if sp == 1:
            return ops.linear_gated_residual(x, w, b, ones, M, resid)
        return ops.linear_splitk(x, w, b, ops.EPI_GATED_RESIDUAL, resid, self._workspace(M, w.shape[0], sp), sp,
                                 gate=ones, rows_per_batch=M)


class QwenVLTextModel:
    """``Qwen2_5_VLTextModel`` forward on the HIP path (one prompt at a time: no padding mask)."""

    def __init__(self, config: Optional[TextEncoderConfig] = None, device="cuda", packed_attention: bool = False):
        self.config = config or TextEncoderConfig()
        self.device = torch.device(device)
        self.packed_attention = packed_attention
        c = self.config
        if c.head_dim % 64 or c.hidden_size % 64 or c.intermediate_size % 64:
            raise NotImplementedError("head_dim, hidden_size and intermediate_size must be multiples of 64")
        if sum(c.mrope_section) * 2 != c.head_dim:
            raise ValueError("mrope_section must cover head_dim / 2")
        self.layers: List[Dict[str, torch.Tensor]] = []
        self.w: Dict[str, torch.Tensor] = {}
        self.lin = EncoderLinears(self.device)
        self.turns, self.axis = section_turns(c.mrope_section, c.rope_theta, self.device)

    # ------------------------------------------------------------------ weights
    @staticmethod
    def _strip(sd: Dict[str, torch.Tensor]) -> Dict[str, torch.Tensor]:
        """Accept the text model's own names and the checkpoint prefixes around it."""
        for pre in ("model.language_model.", "language_model.model.", "language_model.", "model."):
            if any(k.startswith(pre + "layers.") for k in sd):
                return {k[len(pre):]: v for k, v in sd.items() if k.startswith(pre)}
        return sd

    def load_state_dict(self, sd: Dict[str, torch.Tensor]) -> "QwenVLTextModel":
        sd = self._strip(sd)
        c, dev = self.config, self.device
        g = lambda k: sd[k].to(dev).to(BF16).contiguous()  # noqa: E731
        if tuple(sd["embed_tokens.weight"].shape) != (c.vocab_size, c.hidden_size):
            raise ValueError("embed_tokens shape does not match the config")
        self.w = {"embed": g("embed_tokens.weight"), "norm": g("norm.weight"),
                  "ones": torch.ones(1, c.hidden_size, dtype=BF16, device=dev),
                  "zero_d": torch.zeros(c.hidden_size, dtype=BF16, device=dev),
                  "zero_hd": torch.zeros(c.head_dim, dtype=BF16, device=dev),
                  "zero_2f": torch.zeros(2 * c.intermediate_size, dtype=BF16, device=dev)}
        self.layers = []
        for i in range(c.num_hidden_layers):
            p = f"layers.{i}."
            a = p + "self_attn."
            self.layers.append({
                "ln1": g(p + "input_layernorm.weight"), "ln2": g(p + "post_attention_layernorm.weight"),
                "w_qkv": torch.cat([g(a + "q_proj.weight"), g(a + "k_proj.weight"), g(a + "v_proj.weight")]).contiguous(),
                "b_qkv": torch.cat([g(a + "q_proj.bias"), g(a + "k_proj.bias"), g(a + "v_proj.bias")]).contiguous(),
                "w_o": g(a + "o_proj.weight"),
                "w_gu": torch.cat([g(p + "mlp.gate_proj.weight"), g(p + "mlp.up_proj.weight")]).contiguous(),
                "w_down": g(p + "mlp.down_proj.weight"),
            })
        return self

    # ------------------------------------------------------------------ forward
    def forward(self, input_ids: Optional[torch.Tensor] = None, position_ids: Optional[torch.Tensor] = None,
                inputs_embeds: Optional[torch.Tensor] = None) -> torch.Tensor:
        """input_ids [S] (or inputs_embeds [S, D] bf16, e.g. text embeddings with the vision rows
        spliced in), position_ids [3, S] (default: 0..S-1 on all three axes) -> last hidden state
        after the final norm, [S, D] bf16."""
        c, w, dev = self.config, self.w, self.device
        if not self.layers:
            raise RuntimeError("text encoder weights not loaded")
        if self.packed_attention:
            return self.forward_packed([input_ids if inputs_embeds is None else inputs_embeds],
                                       None if position_ids is None else [position_ids])[0]
        D, H, Hk, Dh, F = c.hidden_size, c.num_attention_heads, c.num_key_value_heads, c.head_dim, c.intermediate_size
        S = int(input_ids.numel()) if inputs_embeds is None else int(inputs_embeds.shape[0])
        Sp = -(-S // 64) * 64  # padded rows: GEMM N / K alignment; causal masking keeps rows < S exact
        if position_ids is None:
            position_ids = torch.arange(S).view(1, S).expand(3, S)
        pos = torch.zeros(3, Sp, dtype=torch.long)
        pos[:, :S] = position_ids.cpu()
        cos, sin = (t.to(dev).contiguous() for t in mrope_tables(c, pos))
        x = torch.zeros(Sp, D, dtype=BF16, device=dev)
        if inputs_embeds is None:
            ids = torch.zeros(Sp, dtype=torch.int32, device=dev)
            ids[:S] = input_ids.reshape(-1).to(dev).to(torch.int32)
            ops.embed_rows(w["embed"], ids, out=x)
        else:
            x[:S] = inputs_embeds.to(dev).to(BF16)
        h = torch.empty(Sp, D, dtype=BF16, device=dev)
        qkv = torch.empty(Sp, (H + 2 * Hk) * Dh, dtype=BF16, device=dev)
        att = torch.empty(Sp, H * Dh, dtype=BF16, device=dev)
        s = torch.empty(H * Sp, Sp, dtype=torch.float32, device=dev)  # all heads' scores
        p = torch.empty(H * Sp, Sp, dtype=BF16, device=dev)
        vt = torch.empty(Hk * Dh, Sp, dtype=BF16, device=dev)
        causal = torch.stack([torch.zeros(Sp, dtype=torch.int32), torch.arange(1, Sp + 1, dtype=torch.int32)], 1)
        causal = causal.to(dev)
        gu = torch.empty(Sp, 2 * F, dtype=BF16, device=dev)
        a = torch.empty(Sp, F, dtype=BF16, device=dev)
        scale = 1.0 / math.sqrt(Dh)
        G = H // Hk  # query heads per kv head
        for L in self.layers:
            ops.rmsnorm(x, L["ln1"], out=h, eps=c.rms_norm_eps)
            self.lin.linear(h, L["w_qkv"], L["b_qkv"], qkv)
            ops.rope_half(qkv, 0, H + Hk, Dh, cos, sin)  # q heads, then the k heads right after them
            ops.transpose(qkv[:, (H + Hk) * Dh:], out=vt)  # V^T of every kv head
            # every head in one launch per step: scores, causal softmax, P.V (kv head = q head // G)
            ops.matmul_heads(qkv[:, :Dh], Dh, qkv[:, H * Dh:(H + 1) * Dh], Dh, s[:Sp], Sp * Sp, H, group=G)
            ops.softmax_rows(s, scale, out=p, ranges=causal)
            ops.matmul_heads(p[:Sp], Sp * Sp, vt[:Dh], Dh * Sp, att[:, :Dh], Dh, H, group=G, bias=w["zero_hd"])
            self.lin.residual(att, L["w_o"], w["zero_d"], w["ones"], x)
            ops.rmsnorm(x, L["ln2"], out=h, eps=c.rms_norm_eps)
            self.lin.linear(h, L["w_gu"], w["zero_2f"], gu)
            ops.silu_mul(gu, out=a)
            self.lin.residual(a, L["w_down"], w["zero_d"], w["ones"], x)
        ops.rmsnorm(x, w["norm"], out=h, eps=c.rms_norm_eps)
        return h[:S]

    __call__ = forward

    # ------------------------------------------------------------------ several prompts, new tokens
    def new_cache(self, pages: int, page_size: int = 64) -> PagedKVCache:
        """An empty cache of this model's layers (``extend``)."""
        c = self.config
        return PagedKVCache(c.num_hidden_layers, c.num_key_value_heads, c.head_dim, pages, page_size, self.device)

    def forward_packed(self, prompts: Sequence[torch.Tensor],
                       position_ids: Optional[Sequence[torch.Tensor]] = None) -> List[torch.Tensor]:
        """Several prompts in one pass: token ids [S_i] or embeddings [S_i, D] each, positions [3, S_i]
        or [S_i] (default: 0..S_i-1 on all three axes) -> their last hidden states [S_i, D], as ``forward`` of each."""
        lens = [int(p.shape[0]) if p.is_floating_point() else int(p.numel()) for p in prompts]
        if position_ids is None:
            position_ids = [torch.arange(n).view(1, n).expand(3, n) for n in lens]
        position_ids = self._axes_positions(position_ids, lens)
        cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(self.device)
        H, Hk, Dh = self.config.num_attention_heads, self.config.num_key_value_heads, self.config.head_dim

        def attend(layer, qkv, q3, pos, out):
            ops.rope_axes(qkv, 0, H + Hk, Dh, pos, self.turns, self.axis)
            kv = qkv[:, H * Dh:].unflatten(1, (2, Hk, Dh))
            ops.attention_packed(q3, kv[:, 0], kv[:, 1], cu, out=out)

        return list(self._rows(prompts, position_ids, lens, attend).split(lens))

    def extend(self, cache: PagedKVCache, seqs: Sequence[int], tokens: Sequence[torch.Tensor],
               position_ids: Optional[Sequence[torch.Tensor]] = None) -> List[torch.Tensor]:
        """New tokens (ids [n_i] or embeddings [n_i, D]) of sequences of ``cache``, behind what it holds of
        them: their last hidden states [n_i, D], as the rows that ``forward`` of the whole sequences gives.
        positions [3, n_i] (default: counted on from the sequence's length)."""
        lens = [int(p.shape[0]) if p.is_floating_point() else int(p.numel()) for p in tokens]
        if position_ids is None:
            position_ids = [torch.arange(cache.length(s), cache.length(s) + n).view(1, n).expand(3, n)
                            for s, n in zip(seqs, lens)]
        position_ids = self._axes_positions(position_ids, lens)
        st = cache.step(seqs, lens)
        c = self.config
        H, Hk, Dh = c.num_attention_heads, c.num_key_value_heads, c.head_dim
        try:
            nb = ops.attention_paged_workspace_bytes(sum(lens), len(lens), H, Hk, Dh, st.page_table.shape[1], cache.page_size)
            ws = torch.empty(nb, dtype=torch.uint8, device=self.device) if nb else None

            def attend(layer, qkv, q3, pos, out):
                k, v = cache.k[layer], cache.v[layer]
                ops.rope_append(qkv, H, Hk, Dh, pos, self.turns, self.axis, k, v, st.slots)
                ops.attention_paged(q3, k, v, st.page_table, st.kv_lens, cu_seqlens=st.cu_seqlens, out=out, workspace=ws)

            return list(self._rows(tokens, position_ids, lens, attend).split(lens))
        except Exception:
            cache.take_back(seqs, lens)  # their k / v may be missing
            raise

    def _axes_positions(self, position_ids, lens) -> List[torch.Tensor]:
        """[3, n] each; one row serves all three axes."""
        if not self.layers:
            raise RuntimeError("text encoder weights not loaded")
        if len(position_ids) != len(lens) or any(tuple(p.shape) not in ((3, n), (1, n), (n,)) for p, n in zip(position_ids, lens)):
            raise ValueError("positions [3, tokens], or [tokens] for all three axes, for each sequence")
        return [p.cpu().expand(3, n) for p, n in zip(position_ids, lens)]

    def _rows(self, prompts, position_ids, lens, attend) -> torch.Tensor:
        """The layers over the rows of all sequences, one behind the other; ``attend(layer, qkv, q, positions, out)``
        rotates the rows' heads and fills out [T, H, Dh]."""
        c, w, dev = self.config, self.w, self.device
        D, H, Hk, Dh, F = c.hidden_size, c.num_attention_heads, c.num_key_value_heads, c.head_dim, c.intermediate_size
        T = sum(lens)
        h = torch.empty(T, D, dtype=BF16, device=dev)
        if T == 0:
            return h
        pos = torch.cat(list(position_ids), 1).to(torch.int32).to(dev)
        x = torch.empty(T, D, dtype=BF16, device=dev)
        at = 0
        for p, n in zip(prompts, lens):
            if p.is_floating_point():
                x[at:at + n] = p.to(dev).to(BF16)
            elif n:
                ops.embed_rows(w["embed"], p.reshape(-1).to(dev).to(torch.int32), out=x[at:at + n])
            at += n
        qkv = torch.empty(T, (H + 2 * Hk) * Dh, dtype=BF16, device=dev)
        att = torch.empty(T, H * Dh, dtype=BF16, device=dev)
        q3, out = qkv[:, :H * Dh].unflatten(1, (H, Dh)), att.view(T, H, Dh)
        gu = torch.empty(T, 2 * F, dtype=BF16, device=dev)
        a = torch.empty(T, F, dtype=BF16, device=dev)
        for i, L in enumerate(self.layers):
            ops.rmsnorm(x, L["ln1"], out=h, eps=c.rms_norm_eps)
            self.lin.linear(h, L["w_qkv"], L["b_qkv"], qkv)
            attend(i, qkv, q3, pos, out)
            self.lin.residual(att, L["w_o"], w["zero_d"], w["ones"], x)
            ops.rmsnorm(x, L["ln2"], out=h, eps=c.rms_norm_eps)
            self.lin.linear(h, L["w_gu"], w["zero_2f"], gu)
            ops.silu_mul(gu, out=a)
            self.lin.residual(a, L["w_down"], w["zero_d"], w["ones"], x)
        return ops.rmsnorm(x, w["norm"], out=h, eps=c.rms_norm_eps)


# ---------------------------------------------------------------------------- text + vision
def rope_index(input_ids: torch.Tensor, image_token_id: int, image_grid_thw=None, spatial_merge_size: int = 2
               ) -> torch.Tensor:
    """3-D positions [3, S] for one prompt (Qwen2_5_VLModel.get_rope_index, images only): text runs
    count up on all three axes; an image block of (t, h/m, w/m) merged tokens starting at position
    p gets (p, p + row, p + col) (temporal interval 1 for images), and the text after it resumes at
    p + max(h, w) / m."""
    ids = input_ids.reshape(-1).cpu()
    S = ids.numel()
    grids = [tuple(int(v) for v in g) for g in (image_grid_thw.tolist() if torch.is_tensor(image_grid_thw)
                                                 else (image_grid_thw or []))]
    pos = torch.empty(3, S, dtype=torch.long)
    is_img = (ids == image_token_id).tolist()
    i, cur, gi = 0, 0, 0
    while i < S:
        j = i
        while j < S and is_img[j] == is_img[i]:
            j += 1
        if not is_img[i]:
            pos[:, i:j] = torch.arange(cur, cur + j - i)
            cur += j - i
        else:
            if gi >= len(grids):
                raise ValueError("more <|image_pad|> runs than image_grid_thw entries")
            t, h, w = grids[gi]
            gi += 1
            lh, lw = h // spatial_merge_size, w // spatial_merge_size
            n = t * lh * lw
            if j - i != n:
                raise ValueError(f"image token run of {j - i} != {n} merged patches")
            tt = torch.arange(t).view(t, 1, 1).expand(t, lh, lw).reshape(-1)
            hh = torch.arange(lh).view(1, lh, 1).expand(t, lh, lw).reshape(-1)
            ww = torch.arange(lw).view(1, 1, lw).expand(t, lh, lw).reshape(-1)
            pos[0, i:j], pos[1, i:j], pos[2, i:j] = tt + cur, hh + cur, ww + cur
            cur += max(h, w) // spatial_merge_size
        i = j
    return pos


@dataclass
class _Prefix:
    """A prompt whose k / v the cache holds: its tokens, its pictures' key, its last hidden states."""

    ids: torch.Tensor
    key: Optional[tuple]
    hidden: torch.Tensor


class QwenVLEncoder:
    """``Qwen2_5_VLModel`` (vision tower + language model) as the reference's pipeline calls it
    for prompt embeddings: image embeddings scattered over the ``<|image_pad|>`` tokens, 3-D
    positions from rope_index, last hidden state after the final norm (hidden_states[-1])."""

    IMAGE_TOKEN_ID = 151655  # <|image_pad|> in the Qwen2.5-VL vocabulary

    def __init__(self, text_config: Optional[TextEncoderConfig] = None, vision_config=None, device="cuda",
                 image_token_id: int = IMAGE_TOKEN_ID, vision_cache_size: int = 8, packed_attention: bool = False,
                 prefix_cache_size: int = 0, prefix_cache_pages: Optional[int] = None):
        """``packed_attention``: both models attend without a score matrix in memory, and several prompts
        share a pass (``forward_batch``). ``prefix_cache_size`` > 0: the k / v of the last prompts are kept
        (``prefix_cache_pages`` pages of 64 tokens, default 16 for each and one more), and a prompt that begins like one
        of them -- the template and the same picture -- runs only the tokens behind what they share."""
        from .vision import QwenVLVisionTower, VisionConfig
        self.text = QwenVLTextModel(text_config, device, packed_attention)
        self.vision = QwenVLVisionTower(vision_config or VisionConfig(), device, packed_attention)
        self.prefix_cache_size = prefix_cache_size
        self._prefix_pages = prefix_cache_pages
        self.prefixes: "OrderedDict[int, _Prefix]" = OrderedDict()  # cache sequence -> what it holds
        self.kv: Optional[PagedKVCache] = None
        if self.vision.config.out_hidden_size != self.text.config.hidden_size:
            raise ValueError("vision out_hidden_size must equal the text hidden_size")
        self.image_token_id = image_token_id
        self.device = self.text.device
        # VLM cache (README.md:125,156,182 of the reference: cached_pipeline_v2 / test_vlm_cache):
        # the vision tower's output per condition image, so a prompt change over the same image
        # (the realtime loop's case) re-runs only the language model
        self.vision_cache: "OrderedDict[tuple, torch.Tensor]" = OrderedDict()
        self.vision_cache_size = vision_cache_size

    @property
    def prefix_pages(self) -> int:
        """Pages of the kept prompts' cache, which the first of them makes."""
        return self._prefix_pages or 16 * (self.prefix_cache_size + 1)

    @property
    def packed_attention(self) -> bool:
        """Both models' switch; may be set at any time."""
        return self.text.packed_attention and self.vision.packed_attention

    @packed_attention.setter
    def packed_attention(self, on: bool) -> None:
        self.text.packed_attention = self.vision.packed_attention = bool(on)

    def load_state_dict(self, sd: Dict[str, torch.Tensor]) -> "QwenVLEncoder":
        self.clear_prefixes()
        self.vision_cache.clear()
        self.text.load_state_dict({k: v for k, v in sd.items() if "visual." not in k})
        self.vision.load_state_dict({k: v for k, v in sd.items() if "visual." in k})
        return self

    def forward(self, input_ids: torch.Tensor, pixel_values: Optional[torch.Tensor] = None,
                image_grid_thw=None) -> torch.Tensor:
        """One prompt: input_ids [S] (or [1, S]) -> hidden states [S, D] bf16."""
        if self.prefix_cache_size > 0:
            return self._forward_prefix(input_ids.reshape(-1), pixel_values, image_grid_thw)
        emb, pos = self._embeds(input_ids.reshape(-1), pixel_values, image_grid_thw)
        return self.text(inputs_embeds=emb, position_ids=pos)

    __call__ = forward

    def forward_batch(self, prompts: Sequence[tuple]) -> List[torch.Tensor]:
        """Several prompts, (input_ids, pixel_values or None, image_grid_thw or None) each, in one pass of the
        language model -> their hidden states [S_i, D]."""
        rows = [self._embeds(ids.reshape(-1), pv, grid) for ids, pv, grid in prompts]
        return self.text.forward_packed([e for e, _ in rows], [p for _, p in rows])

    def _embeds(self, ids: torch.Tensor, pixel_values, image_grid_thw):
        """(embeddings [S, D] with the image rows spliced in, positions [3, S]) of one prompt."""
        dev = self.device
        S = ids.numel()
        Sp = -(-S // 64) * 64
        emb = torch.zeros(Sp, self.text.config.hidden_size, dtype=BF16, device=dev)
        ids_dev = torch.zeros(Sp, dtype=torch.int32, device=dev)
        ids_dev[:S] = ids.to(dev).to(torch.int32)
        ops.embed_rows(self.text.w["embed"], ids_dev, out=emb)
        if pixel_values is not None:
            img = self._vision(pixel_values, image_grid_thw)
            where = (ids.cpu() == self.image_token_id).nonzero().view(-1)
            if where.numel() != img.shape[0]:
                raise ValueError(f"{where.numel()} image tokens but {img.shape[0]} image embeddings")
            emb[where.to(dev)] = img  # masked_scatter of the image rows
        return emb[:S], self._positions(ids, pixel_values, image_grid_thw)

    def _positions(self, ids, pixel_values, image_grid_thw) -> torch.Tensor:
        return rope_index(ids, self.image_token_id, image_grid_thw if pixel_values is not None else None,
                          self.vision.config.spatial_merge_size)

    # ------------------------------------------------------------------ prompts that begin alike
    def clear_prefixes(self) -> None:
        """Forget the kept prompts (after a change of weights; load_state_dict does it)."""
        for seq in self.prefixes:
            self.kv.drop(seq)
        self.prefixes.clear()

    def _forward_prefix(self, ids: torch.Tensor, pixel_values, image_grid_thw) -> torch.Tensor:
        ids = ids.cpu()
        S = ids.numel()
        key, rows = None, 0
        image = (ids == self.image_token_id).nonzero().view(-1)
        if pixel_values is not None:
            key, grid = self._vision_key(pixel_values, image_grid_thw)
            rows = sum(t * h * w for t, h, w in grid) // self.vision.config.spatial_merge_size ** 2
        pos = self._positions(ids, pixel_values, image_grid_thw)
        if image.numel() != rows:  # as for a prompt that runs whole, however much of this one is kept
            raise ValueError(f"{image.numel()} image tokens but {rows} image embeddings")
        best, common = None, 0
        for seq, p in reversed(self.prefixes.items()):  # of equals, the one used last
            m = min(S, p.ids.numel())
            ne = (ids[:m] != p.ids[:m]).nonzero()
            n = int(ne[0]) if ne.numel() else m
            if p.key != key and image.numel():  # other pictures: the text before the first one is shared
                n = min(n, int(image[0]))
            if n > common:
                best, common = seq, n
        if best is not None:
            self.prefixes.move_to_end(best)
            if common == S:
                return self.prefixes[best].hidden[:S].clone()  # the caller's own: what is kept stays as it is
        if self.kv is None:
            self.kv = self.text.new_cache(self.prefix_pages)
        kv = self.kv
        # room for the new sequence's pages beside the shared ones; where even all others' would not do, the prompt
        # it begins like goes and it runs whole
        whole = -(-S // kv.page_size)
        need = whole - common // kv.page_size
        if best is not None and kv.num_pages - kv.held_pages(best) < need and whole <= kv.num_pages:
            kv.drop(best)
            del self.prefixes[best]
            best, common, need = None, 0, whole
        while whole <= kv.num_pages and kv.free_pages < need and self.prefixes and next(iter(self.prefixes)) != best:
            old, _ = self.prefixes.popitem(last=False)  # the one used longest ago first
            kv.drop(old)
        if kv.free_pages < need:  # longer than the pool: not kept, and those that are stay
            return self.text.forward_packed([self._embeds(ids, pixel_values, image_grid_thw)[0]], [pos])[0]
        if image.numel() and int(image[-1]) >= common:
            new = self._embeds(ids, pixel_values, image_grid_thw)[0][common:]
        else:
            new = ids[common:]  # every image row lies in what is shared
        seq = self.kv.fork(best, common) if common else self.kv.add()
        try:
            hidden = self.text.extend(self.kv, [seq], [new], [pos[:, common:]])[0]
            if common:
                hidden = torch.cat([self.prefixes[best].hidden[:common], hidden])
            own = hidden.clone()  # the caller's; what is kept stays as it is
        except Exception:
            self.kv.drop(seq)
            raise
        self.prefixes[seq] = _Prefix(ids.clone(), key, hidden)  # the caller may use its buffer again
        while len(self.prefixes) > self.prefix_cache_size:
            old, _ = self.prefixes.popitem(last=False)
            self.kv.drop(old)
        return own

    def _vision_key(self, pixel_values: torch.Tensor, image_grid_thw):
        """(grid and content digest, grid) of a prompt's pictures."""
        grid = tuple(tuple(int(v) for v in g) for g in (image_grid_thw.tolist() if torch.is_tensor(image_grid_thw)
                                                         else image_grid_thw))
        pv = pixel_values.detach().to("cpu", torch.float32).contiguous()
        return (grid, hashlib.blake2b(pv.numpy().tobytes(), digest_size=16).hexdigest()), grid

    def _vision(self, pixel_values: torch.Tensor, image_grid_thw) -> torch.Tensor:
        grid = tuple(tuple(int(v) for v in g) for g in (image_grid_thw.tolist() if torch.is_tensor(image_grid_thw)
                                                         else image_grid_thw))
        if self.vision_cache_size <= 0:
            return self.vision.forward(pixel_values, grid)
        key, _ = self._vision_key(pixel_values, grid)
        hit = self.vision_cache.get(key)
        if hit is not None:
            self.vision_cache.move_to_end(key)
            return hit
        img = self.vision.forward(pixel_values, grid)
        self.vision_cache[key] = img
        while len(self.vision_cache) > self.vision_cache_size:
            self.vision_cache.popitem(last=False)
        return img


def _image_digest(im) -> str:
    """Content key of a condition image (PIL or tensor) for the prompt-embedding cache."""
    if torch.is_tensor(im):
        data = im.detach().contiguous().view(-1).view(torch.uint8).cpu().numpy().tobytes()  # any dtype, bf16 too
        tag = (tuple(im.shape), str(im.dtype))
    else:
        data, tag = im.tobytes(), (im.size, im.mode)
    return hashlib.blake2b(repr(tag).encode() + data, digest_size=16).hexdigest()


# ---------------------------------------------------------------------------- pipeline hook
PROMPT_TEMPLATE = (
    "<|im_start|>system\nDescribe the key features of the input image (color, shape, size, texture, objects, "
    "background), then explain how the user's text instruction should alter or modify the image. Generate a new "
    "image that meets the user's requirements while maintaining consistency with the original input image."
    "<|im_end|>\n<|im_start|>user\n{}<|im_end|>\n<|im_start|>assistant\n")
IMAGE_PROMPT_TEMPLATE = "Picture {}: <|vision_start|><|image_pad|><|vision_end|>"
PROMPT_DROP_TOKENS = 64  # prompt_template_encode_start_idx
CONDITION_IMAGE_AREA = 384 * 384


def condition_size(width: int, height: int, area: int = CONDITION_IMAGE_AREA) -> Tuple[int, int]:
    """calculate_dimensions(area, w / h): w = sqrt(area r), h = w / r, each rounded to 32."""
    r = width / height
    w = math.sqrt(area * r)
    h = w / r
    return int(round(w / 32) * 32), int(round(h / 32) * 32)


class QwenImageEditPromptEncoder:
    """``pipe.prompt_encoder`` for QwenImageEditPlusPipeline (encode_prompt's Edit-Plus
    form): format the template with one "Picture i" prefix per condition image,
    run the processor (tokenizer + Qwen2VLImageProcessor, as the reference does -- its vocabulary
    files come with the checkpoint), encode on the HIP path, drop the first 64 tokens.
    ``processor(text=[str], images=[PIL...], return_tensors="pt")`` must return input_ids,
    pixel_values and image_grid_thw (the HF processor's keys)."""

    def __init__(self, encoder: QwenVLEncoder, processor, drop_tokens: int = PROMPT_DROP_TOKENS,
                 cache_size: int = 32):
        self.encoder, self.processor, self.drop = encoder, processor, drop_tokens
        # prompt-embedding cache keyed by (prompt, condition-image contents): the reference's
        # cached_pipeline (README.md:124) reuse of prompt / image embeddings
        self.cache: "OrderedDict[tuple, tuple]" = OrderedDict()
        self.cache_size = cache_size

    def _condition_images(self, image):
        if image is None:
            return []
        imgs = image if isinstance(image, (list, tuple)) else [image]
        from PIL import Image
        out = []
        for im in imgs:
            if hasattr(im, "resize") and hasattr(im, "size") and not torch.is_tensor(im):
                # Edit-Plus resizes through VaeImageProcessor.resize, whose default is LANCZOS [U]
                w, h = condition_size(*im.size)
                out.append(im.resize((w, h), Image.LANCZOS))
            else:
                out.append(im)
        return out

    def __call__(self, prompt, image=None):
        prompts = [prompt] if isinstance(prompt, str) else list(prompt)
        ims = [] if image is None else (image if isinstance(image, (list, tuple)) else [image])
        key = (tuple(prompts), tuple(_image_digest(im) for im in ims)) if self.cache_size > 0 else None
        if key is not None and key in self.cache:
            self.cache.move_to_end(key)
            return self.cache[key]
        out = self._encode(prompts, image)
        if key is not None:
            self.cache[key] = out
            while len(self.cache) > self.cache_size:
                self.cache.popitem(last=False)
        return out

    def _encode(self, prompts, image):
        imgs = self._condition_images(image)
        prefix = "".join(IMAGE_PROMPT_TEMPLATE.format(i + 1) for i in range(len(imgs)))
        inputs = []
        for p in prompts:
            kw = {"images": imgs} if imgs else {}
            mi = self.processor(text=[PROMPT_TEMPLATE.format(prefix + p)], return_tensors="pt", **kw)
            ids = mi["input_ids"][0]
            if "attention_mask" in mi:
                ids = ids[mi["attention_mask"][0].bool()]
            inputs.append((ids, mi.get("pixel_values"), mi.get("image_grid_thw")))
        enc = self.encoder
        if len(inputs) > 1 and getattr(enc, "packed_attention", False) and not enc.prefix_cache_size:
            rows = enc.forward_batch(inputs)  # one pass over all prompts
        else:
            rows = [enc(*i) for i in inputs]
        rows = [h[self.drop:] for h in rows]
        L = max(r.shape[0] for r in rows)
        D = rows[0].shape[1]
        embeds = torch.zeros(len(rows), L, D, dtype=BF16, device=rows[0].device)
        mask = torch.zeros(len(rows), L, dtype=torch.long, device=rows[0].device)
        for i, r in enumerate(rows):
            embeds[i, :r.shape[0]] = r
            mask[i, :r.shape[0]] = 1
        return embeds, mask
