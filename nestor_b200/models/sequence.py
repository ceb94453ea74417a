"""``SequenceModel(adapter, backbone, head)`` and the ``Model.from_config`` factory.

Parity targets: ``nestor/models/sequence.py:40-179`` (composition, fused head hand-off),
``nestor/adapters/text.py:120-180`` (embedding x ``embedding_multiplier``, trivial-mask
contract: pre-tokenised tensors carry no attention mask), ``nestor/heads/language_modeling.py:85-98``
(``logits = projection(h) * logit_multiplier``).
"""

from __future__ import annotations

import contextlib
import dataclasses as dc
import os
from typing import Any

import torch
from torch import Tensor, nn

from nestor_b200 import ops
from nestor_b200.ops import _lib
from nestor_b200.configs.model import (
    LanguageModelingHeadConfig, NestorConfig, ReferenceMupConfig, SequenceModelConfig, TextAdapterConfig,
)
from nestor_b200.models.modules import LayerStack, Matrix
from nestor_b200.models.nestor import EIGHT_BIT, Nestor, NestorKVCache, W
from nestor_b200.models.registry import (
    ADAPTERS, BACKBONES, HEADS, MODELS, register_adapter, register_backbone, register_head, register_model,
)
from nestor_b200.models.scaling import _ACTIVATIONS as SCALING_ACTIVATIONS, RMSNorm, ScaledLinear
from nestor_b200.models.tags import ADAMW_DECAY, ParamTag, tag


@dc.dataclass
class ModelOutput:
    """``pred``: logits ``[B, S, V]`` — or the head input ``[B, S, d]`` when the head is fused
    into the loss — and ``aux``: routing indices per block plus the fused-head handle."""

    pred: Tensor
    aux: dict[str, Any]


class ByteTokenizer:
    """UTF-8 bytes as token ids (``tokenizer="bytes"``): needs no vocabulary file, for tests and offline use."""

    n_vocab = 256

    def encode_ordinary(self, text: str) -> list[int]:
        return list(text.encode("utf-8"))

    def decode(self, ids: list[int]) -> str:
        return bytes(int(i) & 0xFF for i in ids).decode("utf-8", errors="replace")


@register_adapter(TextAdapterConfig)
class TextAdapter(nn.Module):
    """Token embedding table; output ``norm(E[ids]) * embedding_multiplier`` in fp32.

    Without a reference-muP recipe the embeddings are normalised to unit RMS (learned gain) before the first block, as
    in the reference's adapter (``nestor/adapters/text.py:71-75,150``); the recipe replaces that norm by the identity
    and scales by its embedding multiplier instead (``nestor/scaling/reference_mup.py:320``).

    The adapter is also the tokenizer for string inputs (reference ``nestor/adapters/text.py:59-101``): a tiktoken
    encoding named by ``config.tokenizer`` (loaded lazily; pre-tokenised tensors never need it), or the built-in
    ``"bytes"`` tokenizer. ``encode_texts`` right-pads a batch to its longest entry (capped at ``max_length``) and
    returns the validity mask; pre-tokenised tensors carry no mask (every position is a real token).
    """

    def __init__(self, config: TextAdapterConfig, mup: ReferenceMupConfig | None) -> None:
        super().__init__()
        if config.vocab_size is None:
            raise ValueError("TextAdapterConfig.vocab_size is required (token ids are the only input form).")
        self.config = config
        self.embed = nn.Embedding(config.vocab_size, config.embed_dim)
        tag(self.embed.weight, ADAMW_DECAY)
        std = mup.initializer_range if mup is not None else 1.0
        nn.init.normal_(self.embed.weight, 0.0, std)
        self.embedding_multiplier = mup.embedding_multiplier if mup is not None else 1.0
        self.norm = RMSNorm(config.embed_dim) if mup is None else None
        self._tokenizer: Any = None

    def tokenizer(self) -> Any:
        if self._tokenizer is None:
            if self.config.tokenizer == "bytes":
                self._tokenizer = ByteTokenizer()
            else:
                try:
                    import tiktoken
                    self._tokenizer = tiktoken.get_encoding(self.config.tokenizer)
                except Exception as exc:   # no package, or no vocabulary file on a machine without network
                    raise RuntimeError(f"cannot load the {self.config.tokenizer!r} tokenizer for string inputs: {exc}. "
                                       "Pass token-id tensors, or use tokenizer='bytes'.") from exc
        return self._tokenizer

    def encode_texts(self, texts: list[str], device: torch.device | None = None) -> tuple[Tensor, Tensor]:
        """``(ids [B, L] int64, valid [B, L] bool)`` for a batch of strings, right-padded with id 0."""

        tok = self.tokenizer()
        rows = [tok.encode_ordinary(t)[: self.config.max_length] for t in texts]
        if any(max(r, default=0) >= self.embed.num_embeddings for r in rows):
            raise ValueError("the tokenizer produced an id beyond the embedding table")
        L = max(1, max(len(r) for r in rows))
        ids = torch.zeros(len(rows), L, dtype=torch.long)
        valid = torch.zeros(len(rows), L, dtype=torch.bool)
        for i, r in enumerate(rows):
            ids[i, : len(r)] = torch.tensor(r, dtype=torch.long)
            valid[i, : len(r)] = True
        device = self.embed.weight.device if device is None else device
        return ids.to(device), valid.to(device)

    def forward(self, ids: Tensor) -> Tensor:
        x = self.embed(ids).float()
        if self.norm is not None:
            x = self.norm(x)
        return x * self.embedding_multiplier


@register_head(LanguageModelingHeadConfig)
class LanguageModelingHead(nn.Module):
    """Unembedding ``[V, d]``, optionally behind hidden layers; ``logit_multiplier = 1 / width_multiplier`` under muP.

    ``hidden_dims`` (usually empty) inserts in-stream layers with ``activation`` between the backbone features and the
    vocabulary matrix (reference ``nestor/heads/language_modeling.py:70-76``). They run as ``pre``; the vocabulary
    matrix stays a single ``[V, d_last]`` weight so that the fused head + cross-entropy kernel path applies to it
    unchanged.
    """

    def __init__(self, config: LanguageModelingHeadConfig, dim: int, mup: ReferenceMupConfig | None) -> None:
        super().__init__()
        dims = [dim, *config.hidden_dims]
        self.hidden = nn.ModuleList(ScaledLinear(a, b, role="in_stream") for a, b in zip(dims[:-1], dims[1:]))
        if config.activation not in SCALING_ACTIVATIONS:
            raise ValueError(f"Unknown head activation {config.activation!r}.")
        self.activation = config.activation
        last = dims[-1]
        std = mup.initializer_range if mup is not None else 1.0 / last
        self.projection = LayerStack([Matrix(last, config.vocab_size, ADAMW_DECAY, std)])
        self.logit_multiplier = 1.0 / mup.width_multiplier if mup is not None else 1.0
        self.vocab_size = config.vocab_size

    @property
    def weight(self) -> Tensor:
        return self.projection.layers[0].weight

    def pre(self, h: Tensor) -> Tensor:
        """The hidden layers in front of the vocabulary matrix (identity for the usual single-matrix head)."""

        act = SCALING_ACTIVATIONS[self.activation]
        for layer in self.hidden:
            h = act(layer(h.to(layer.weight.dtype)))
        return h

    def forward(self, h: Tensor, cd: torch.dtype) -> Tensor:
        return (self.pre(h).to(cd) @ W(self, self.weight).to(cd).t()) * self.logit_multiplier


register_backbone(NestorConfig)(lambda config, mup, **kw: Nestor(config, mup, **kw))


def apply_recipe_variants(model: nn.Module, mup: ReferenceMupConfig) -> None:
    """Optimizer-tag variants of the reference-muP recipe (``nestor/scaling/reference_mup.py:126-311``).

    The models are built with the tags of the Muon pairing (in-stream matrices Muon, single-matrix routers and path
    gates AdamW at the base rate). This pass applies what differs from it:

    * ``matrix_optimizer="adamw"``: attention and expert matrices move to AdamW at ``1 / width_multiplier`` of the base
      rate; routers follow them unless ``NESTOR_MUP_ROUTER_BASE_LR=1`` keeps them at the base rate (the reference
      transform never marks a router); path gates take the matrix rate. The group router's hidden layers stay Muon.
    * ``group_router_lr="base"``: the group router's score / noise read-outs train at the base AdamW rate instead of
      ``score_lr_mul / hidden``.
    * ``NESTOR_MUP_ROUTER_BASE_INIT=1``: single-matrix routers are re-drawn at ``initializer_range`` instead of
      ``initializer_range / sqrt(width_multiplier)``.
    """

    if not mup.enabled("optimizer"):
        return
    muon_matrices = mup.matrix_optimizer == "muon"
    matrix_lr_mul = 1.0 / mup.width_multiplier
    router_lr_mul = 1.0 if muon_matrices or os.environ.get("NESTOR_MUP_ROUTER_BASE_LR", "0") == "1" else matrix_lr_mul
    router_init = os.environ.get("NESTOR_MUP_ROUTER_BASE_INIT", "0") == "1" and mup.enabled("initialization")

    def adamw(p: Tensor, lr_mul: float) -> None:
        tag(p, ParamTag("adamw", lr_mul=lr_mul, weight_decay=True))

    def router(r) -> None:
        w = r.score_mlp.layers[0].weight
        if len(r.score_mlp.layers) == 1:
            adamw(w, router_lr_mul)
            if router_init:
                with torch.no_grad():
                    w.normal_(0.0, mup.initializer_range)

    for block in model.backbone.blocks:
        for layer in block.layers:
            if not muon_matrices:
                for g in layer.attention_groups:
                    for lin in (g.q_proj, g.k_proj, g.v_proj, g.out_proj):
                        adamw(lin.weight, matrix_lr_mul)
                banks = [b for b in (layer.stacked_moe_bank,) if b is not None]
                if layer.expert_pool is not None:
                    banks += [b for b in (layer.expert_pool.stacked_public, layer.expert_pool.stacked_private) if b is not None]
                for bank in banks:
                    for w in bank.matrices():
                        adamw(w, matrix_lr_mul)
                for expert in [*(layer.shared_experts or []), *layer.dense_shared_experts]:
                    for lin in expert.matrices():
                        adamw(lin.weight, matrix_lr_mul)
            if layer.expert_router is not None:
                router(layer.expert_router)
            pool = layer.expert_pool
            if pool is not None:
                for r in ([pool.public_router] if pool.public_router is not None else []) + list(pool.private_routers):
                    router(r)
                if pool.path_gate is not None:
                    adamw(pool.path_gate.weight, router_lr_mul if muon_matrices else matrix_lr_mul)
        if mup.group_router_lr == "base" and block.spec.G > 1:
            for mlp in (block.group_router.score_mlp, block.group_router.noise_mlp):
                if mlp is not None:
                    adamw(mlp.layers[-1].weight, 1.0)


@contextlib.contextmanager
def _evaluating(*models: nn.Module):
    """The models in evaluation mode, and as they were behind it, however it is left."""

    was = [m.training for m in models]
    for m in models:
        m.eval()
    try:
        yield
    finally:
        for m, training in zip(models, was):
            m.train(training)


def _check_kernels(cache) -> None:
    """Raise if a kernel of an 8-bit decode state has reported a failure (reads one word, so it waits for the step)."""

    if getattr(cache, "kernels", False):
        _lib.check_status(cache.positions.device)


@register_model(SequenceModelConfig)
class SequenceModel(nn.Module):
    """adapter -> backbone -> head, each built from its config through the registries.

    ``fused_head=True`` (the training default) returns the normalised head input as ``pred``
    and exposes the head through ``aux["fused_head_module"]`` so the loss can run the
    chunked head+cross-entropy without materialising ``[T, V]`` logits.
    """

    def __init__(self, config: SequenceModelConfig) -> None:
        super().__init__()
        self.config = config
        mup = config.reference_mup
        if config.adapter_config.embed_dim != config.backbone_config.input_dim:
            raise ValueError("adapter embed_dim must equal backbone input_dim.")
        dense_no_router = os.environ.get("NESTOR_DENSE_NO_ROUTER", "1") == "1"
        self.adapter = ADAPTERS.build(config.adapter_config, mup)
        self.backbone = BACKBONES.build(config.backbone_config, mup, dense_no_router=dense_no_router)
        self.head = HEADS.build(config.head_config, self.backbone.output_dim, mup)
        if mup is not None:
            apply_recipe_variants(self, mup)
        self.fused_head = False
        self.compute_dtype: torch.dtype | None = None
        # NESTOR_FASTPATH_CHECK=1: the first three kernel-path forwards are repeated on the PyTorch statement of the
        # ops with the same routing and the largest difference is printed (reference nestor/backbones/nestor.py:4868-4884)
        self._fastpath_checks = 3 if os.environ.get("NESTOR_FASTPATH_CHECK") == "1" else 0

    def resolve_compute_dtype(self, device: torch.device) -> torch.dtype:
        if self.compute_dtype is not None:
            return self.compute_dtype
        return torch.bfloat16 if device.type == "cuda" else torch.float32

    def forward(self, ids: Tensor | list[str], pos: Tensor | None = None, noises: list | None = None,
                valid: Tensor | None = None) -> ModelOutput:
        """``ids``: token ids ``[B, S]`` or a list of strings (tokenised by the adapter, right-padded).

        ``valid [B, S]`` marks real tokens of right-padded batches. The decoder is causal, so padding after a
        sequence cannot reach any valid position; the mask only has to keep padding out of what is *counted*: it is
        handed on as ``aux["valid_token_mask"]``, which the loss (targets), the router statistics (loss-free
        balancing, auxiliary losses) and the evaluation metrics honour. Padding must follow the real tokens.
        """

        if isinstance(ids, (list, tuple)) and ids and isinstance(ids[0], str):
            ids, valid = self.adapter.encode_texts(list(ids))
        if valid is not None and bool((valid[:, 1:] & ~valid[:, :-1]).any()):
            raise ValueError("valid_token_mask must be a prefix mask (padding only after the real tokens).")
        if valid is not None and not getattr(self.backbone.config, "causal", True) and not bool(valid.all()):
            raise ValueError("a bidirectional (causal=False) model attends to every position of its sequence: "
                             "padded batches are not supported, pass sequences of equal length")
        B, S = ids.shape
        cd = self.resolve_compute_dtype(ids.device)
        x0 = self.adapter(ids).reshape(B * S, -1)
        if valid is not None:
            x0 = x0 * valid.reshape(B * S, 1).to(x0.dtype)
        if ids.is_cuda and cd != torch.bfloat16 and ops.use_kernels(ids):
            # the kernels compute in bf16; a full-precision forward on a GPU is the PyTorch statement of every op
            with ops.oracle_ops():
                h, aux = self.backbone(x0, B, S, cd, pos=pos, noises=noises)
        elif self._fastpath_checks > 0 and ops.use_kernels(ids) and not torch.cuda.is_current_stream_capturing():
            h, aux = self._checked_forward(x0, B, S, cd, pos, noises)
        else:
            h, aux = self.backbone(x0, B, S, cd, pos=pos, noises=noises)
        if valid is not None:
            aux["valid_token_mask"] = valid
            aux["input_ids"] = ids
            flat = valid.reshape(-1)
            for block in aux["blocks"]:          # the routers' own records carry the mask too
                if "group_router" in block:
                    block["group_router"]["valid_token_mask"] = flat
                for layer in block["layers"]:
                    if "expert_router" in layer:
                        layer["expert_router"]["valid_token_mask"] = flat
        if self.fused_head:
            aux["fused_head_module"] = self.head
            return ModelOutput(pred=self.head.pre(h).view(B, S, -1), aux=aux)
        return ModelOutput(pred=self.head(h, cd).view(B, S, -1), aux=aux)

    def _checked_forward(self, x0: Tensor, B: int, S: int, cd: torch.dtype, pos, noises):
        """Kernel-path forward followed by the same forward on the PyTorch ops, with the first pass's routing replayed
        and the same router noise; prints ``[FASTPATH-CHECK] max|kernels - oracle|`` of the head input."""

        self._fastpath_checks -= 1
        if noises is None and self.training:
            noises = [torch.randn(x0.shape[0], b.spec.G, device=x0.device) if b.spec.G > 1 else None
                      for b in self.backbone.blocks]
        tape = ops.RoutingTape()
        ops.set_routing_tape(tape, "record")
        try:
            h, aux = self.backbone(x0, B, S, cd, pos=pos, noises=noises)
            ops.set_routing_tape(tape, "replay")
            with torch.no_grad(), ops.oracle_ops():
                h_ref, _ = self.backbone(x0.detach(), B, S, cd, pos=pos, noises=noises)
        finally:
            ops.set_routing_tape(None)
        diff = (h.detach().float() - h_ref.float()).abs().max().item()
        print(f"[FASTPATH-CHECK] max|kernels - oracle| = {diff:.3e} (head input, {x0.shape[0]} tokens)", flush=True)
        return h, aux

    # ------------------------------------------------------------------ incremental decoding
    def init_kv_cache(self, batch_size: int, max_len: int, device=None, dtype: torch.dtype = torch.float32):
        """Empty decode state. ``dtype`` int8 or float8_e4m3fn keeps keys and values in 8 bits (``ops.kv8_attention``) and
        lets a step feed several tokens at once."""

        device = self.head.weight.device if device is None else device
        if dtype not in EIGHT_BIT:      # (all that a backbone's own decode state has to take)
            return self.backbone.init_kv_cache(batch_size, max_len, device, dtype)
        return self.backbone.init_kv_cache(batch_size, max_len, device, dtype, open_dtype=self._step_dtype(torch.device(device)))

    def _step_dtype(self, device: torch.device) -> torch.dtype:
        return torch.float32 if self.compute_dtype is None or device.type != "cuda" else self.compute_dtype

    @torch.no_grad()
    def decode_step(self, ids: Tensor, cache, pos: Tensor | None = None) -> Tensor:
        """Logits ``[B, V]`` of the next position given the new tokens ``ids [B]`` or ``[B, 1]`` (``cache`` is advanced).
        Several tokens ``ids [B, n]`` give ``[B, n, V]``, the logits after each of them: one pass over an 8-bit cache, ``n``
        single steps otherwise. An fp32 state may be stepped with fewer sequences than it holds, the first of them. The
        decode state of a backbone other than ``Nestor`` needs no more than a ``length``, the tokens fed so far."""

        eight_bit, batch = getattr(cache, "eight_bit", False), getattr(cache, "batch", ids.shape[0])
        if ids.shape[0] > batch or (eight_bit and ids.shape[0] != batch):
            raise ValueError(f"the cache decodes {batch} sequences, got tokens for {ids.shape[0]}")
        if ids.dim() == 2 and ids.shape[1] == 1:
            ids, pos = ids[:, 0], None if pos is None else pos.reshape(-1)
        if ids.dim() == 2:
            if not eight_bit:
                steps = [self.decode_step(ids[:, t], cache, None if pos is None else pos[:, t]) for t in range(ids.shape[1])]
                return torch.stack(steps, dim=1) if steps else ids.new_zeros(*ids.shape, self.head.vocab_size, dtype=torch.float32)
            if ids.shape[1] == 0:
                return ids.new_zeros(*ids.shape, self.head.vocab_size, dtype=torch.float32)
        cd = self._step_dtype(ids.device)
        return self.head(self._step(ids, cache, pos, cd), cd).float().view(*ids.shape, -1)

    def _step(self, ids: Tensor, cache, pos: Tensor | None, cd: torch.dtype) -> Tensor:
        """The head's input for the new tokens ``ids [B]`` or ``[B, n]``, a row for each (``cache`` is advanced)."""

        B = ids.shape[0]
        rows = ids.reshape(B, -1)
        if pos is None:
            at = getattr(cache, "positions", None)
            at = torch.full((B,), cache.length, dtype=torch.long, device=ids.device) if at is None else at[:B]
            pos = at.unsqueeze(1) + torch.arange(rows.shape[1], device=ids.device)
            pos = pos if ids.dim() == 2 else pos.squeeze(1)
        x0 = self.adapter(rows).reshape(rows.numel(), -1)
        h, _ = self.backbone.forward_step(x0, pos, cache, cd)
        return h

    def _prefill(self, prompt: Tensor, cache) -> Tensor | None:
        """Feed ``prompt [B, S]`` and return the logits after its last token (``None`` for an empty prompt): pieces of up to
        ``PREFILL`` tokens into an 8-bit cache, token by token otherwise. (A piece asks the head for its last row alone: the
        logits of 512 tokens of 64 sequences would take 13 GB.)"""

        B, S = prompt.shape
        if S == 0:
            return None
        if not getattr(cache, "eight_bit", False):
            for t in range(S):
                logits = self.decode_step(prompt[:, t], cache)
            return logits
        cd = self._step_dtype(prompt.device)
        for a in range(0, S, self.PREFILL):
            h = self._step(prompt[:, a : a + self.PREFILL], cache, None, cd)
        return self.head(h.view(B, -1, h.shape[-1])[:, -1].contiguous(), cd).float()

    PREFILL = 512

    @torch.no_grad()
    def generate(self, prompt: Tensor, max_new_tokens: int, temperature: float = 0.0,
                 generator: torch.Generator | None = None, cache_dtype: torch.dtype = torch.float32,
                 draft: "SequenceModel | None" = None, draft_tokens: int = 4) -> Tensor:
        """Greedy (``temperature == 0``) or sampled continuation of ``prompt [B, S0]``; returns ``[B, S0 + new]``.

        ``cache_dtype`` int8 or float8_e4m3fn decodes over an 8-bit cache. With ``draft`` (a smaller model over the same
        vocabulary) each round lets it propose ``draft_tokens`` tokens, scores them in one pass over an 8-bit cache and
        keeps the prefix that :func:`ops.verify_draft` accepts plus one token drawn from what is left: greedy output is
        this model's own, sampled output has its distribution, up to the arithmetic of the cache.
        """

        if draft is not None:
            with _evaluating(self, draft):
                return self._generate_with_draft(prompt, max_new_tokens, temperature, generator, cache_dtype, draft, draft_tokens)
        with _evaluating(self):
            return self._generate(prompt, max_new_tokens, temperature, generator, cache_dtype)

    def _generate(self, prompt: Tensor, max_new_tokens: int, temperature: float, generator: torch.Generator | None,
                  cache_dtype: torch.dtype) -> Tensor:
        B, S0 = prompt.shape
        cache = self.init_kv_cache(B, S0 + max_new_tokens, prompt.device, cache_dtype)
        logits = self._prefill(prompt, cache)
        out = [prompt]
        for i in range(max_new_tokens):
            _check_kernels(cache)          # (before a draw from what they left, which may be NaN)
            if temperature > 0:
                nxt = torch.multinomial(torch.softmax(logits / temperature, dim=-1), 1, generator=generator).squeeze(1)
            else:
                nxt = logits.argmax(dim=-1)
            out.append(nxt.unsqueeze(1))
            logits = self.decode_step(nxt, cache)
        _check_kernels(cache)
        return torch.cat(out, dim=1)

    def _generate_with_draft(self, prompt: Tensor, max_new_tokens: int, temperature: float, generator: torch.Generator | None,
                             cache_dtype: torch.dtype, draft: "SequenceModel", n: int) -> Tensor:
        if draft.head.vocab_size != self.head.vocab_size:
            raise ValueError(f"the draft model has a vocabulary of {draft.head.vocab_size} tokens, this one of {self.head.vocab_size}")
        B, S0 = prompt.shape
        most = NestorKVCache.TAKE_BACK
        if not 1 <= n < most:
            raise ValueError(f"draft_tokens must be in 1..{most - 1} (a refused round has to be taken back), got {n}")
        if S0 < 1:
            raise ValueError("decoding with drafts needs a prompt of at least one token")
        dev = prompt.device
        room = S0 + max_new_tokens + 2 * (n + 1)      # (a sequence may overshoot by a round and then waits, feeding rounds)
        caches = [m.init_kv_cache(B, room, dev, cache_dtype) for m in (self, draft)]
        for m, cache in zip((self, draft), caches):
            if not hasattr(cache, "rollback"):
                raise ValueError(f"decoding with drafts takes tokens back, which the decode state of {type(m.backbone).__name__} does not offer")
        for m, cache in zip((self, draft), caches):
            m._prefill(prompt[:, :-1], cache)
        out = torch.zeros(B, room, dtype=prompt.dtype, device=dev)
        out[:, :S0] = prompt
        end = torch.full((B,), S0, dtype=torch.long, device=dev)             # tokens of each sequence so far
        last = prompt[:, -1]                                                 # the newest of them: not fed yet
        while max_new_tokens > 0 and bool((end < S0 + max_new_tokens).any()):
            tokens, probs, cur = [], [], last
            for i in range(n):
                logits = draft.decode_step(cur, caches[1])
                _check_kernels(caches[1])
                if temperature > 0:
                    probs.append(torch.softmax(logits / temperature, dim=-1))
                    cur = torch.multinomial(probs[-1], 1, generator=generator).squeeze(1)
                else:
                    cur = logits.argmax(dim=-1)
                tokens.append(cur)
            draft.decode_step(cur, caches[1])                                # (the last proposal enters its cache as well)
            x = torch.stack(tokens, dim=1)
            logits = self.decode_step(torch.cat((last.unsqueeze(1), x), dim=1), caches[0])
            _check_kernels(caches[0])
            if temperature > 0:
                target, q = torch.softmax(logits / temperature, dim=-1), torch.stack(probs, dim=1)
            else:
                target, q = torch.zeros_like(logits).scatter_(2, logits.argmax(dim=-1, keepdim=True), 1.0), None
            u = torch.rand(B, n, generator=generator, device=dev)
            w = torch.rand(B, generator=generator, device=dev)
            accepted, token = ops.verify_draft(target, x, q, u, w)
            if bool((token < 0).any()):
                raise RuntimeError("the model's probabilities leave no token to draw (its logits are not finite)")
            accepted, token = accepted.long(), token.to(prompt.dtype)
            # sequences that have their tokens wait for the others: they keep nothing of the round
            live = end < S0 + max_new_tokens
            new = torch.cat((x, token.unsqueeze(1)), dim=1).to(prompt.dtype)
            new.scatter_(1, accepted.unsqueeze(1), token.unsqueeze(1))
            at = torch.arange(n + 1, device=dev).unsqueeze(0)
            keep = live.unsqueeze(1) & (at <= accepted.unsqueeze(1))
            place = end.unsqueeze(1) + at
            out.scatter_(1, place, torch.where(keep, new, out.gather(1, place)))
            kept = torch.where(live, accepted + 1, 0)
            end, last = end + kept, torch.where(live, token, last)
            for cache in caches:
                cache.rollback(n + 1 - kept)
        return out[:, : S0 + max_new_tokens]

    def fsdp2_wrap_order(self) -> list[nn.Module]:
        """Sharding units, in gather order: adapter, each block, backbone tail, head, root."""

        return [self.adapter, *self.backbone.blocks, self.backbone, self.head, self]


class Model:
    """Factory namespace: ``Model.from_config(config)`` builds whatever model is registered for the config's type."""

    @staticmethod
    def from_config(config: Any) -> nn.Module:
        return MODELS.build(config)
