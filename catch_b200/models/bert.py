"""BERT encoder with a sequence-classification head (BERT-base by default:
12 layers, hidden 768, 12 heads, FFN 3072, vocabulary 30522).

The reference lists BERT among the networks it trains
(docs/user_guide/source/pytorch_8_training/Pytorch_training.rst:10-18) with plain
matmul / bmm / softmax eager ops; this definition uses exactly those ops (embedding,
LayerNorm, linear, bmm, softmax, GELU, dropout), all of which have kernels in this
backend.  ``BertConfig.position_embedding_type`` chooses how tokens learn of their places:
``"absolute"`` (embeddings, the default), ``"relative_bias"`` (a learned bias of the scores by
relative position, one table for each layer) or ``"rotary"`` (queries and keys are normalised
and rotated by position).
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn


@dataclass
class BertConfig:
    vocab_size: int = 30522
    hidden_size: int = 768
    num_hidden_layers: int = 12
    num_attention_heads: int = 12
    intermediate_size: int = 3072
    max_position_embeddings: int = 512
    type_vocab_size: int = 2
    hidden_dropout_prob: float = 0.1
    attention_probs_dropout_prob: float = 0.1
    layer_norm_eps: float = 1e-12
    num_labels: int = 2
    position_embedding_type: str = "absolute"   # or "relative_bias", "rotary"
    relative_attention_num_buckets: int = 32
    relative_attention_max_distance: int = 128
    rotary_base: float = 10000.0


class BertEmbeddings(nn.Module):
    absolute = True  # (also for modules that were pickled before there was a choice)

    def __init__(self, c: BertConfig):
        super().__init__()
        self.word_embeddings = nn.Embedding(c.vocab_size, c.hidden_size)
        self.absolute = getattr(c, "position_embedding_type", "absolute") == "absolute"
        if self.absolute:
            self.position_embeddings = nn.Embedding(c.max_position_embeddings, c.hidden_size)
        self.token_type_embeddings = nn.Embedding(c.type_vocab_size, c.hidden_size)
        self.LayerNorm = nn.LayerNorm(c.hidden_size, eps=c.layer_norm_eps)
        self.dropout = nn.Dropout(c.hidden_dropout_prob)
        self.register_buffer("position_ids", torch.arange(c.max_position_embeddings).unsqueeze(0), persistent=False)

    def forward(self, input_ids, token_type_ids=None):
        L = input_ids.shape[1]
        if token_type_ids is None:
            token_type_ids = torch.zeros_like(input_ids)
        if self.absolute:
            x = (self.word_embeddings(input_ids) + self.position_embeddings(self.position_ids[:, :L]) +
                 self.token_type_embeddings(token_type_ids))
        else:
            x = self.word_embeddings(input_ids) + self.token_type_embeddings(token_type_ids)
        return self.dropout(self.LayerNorm(x))


class BertSelfAttention(nn.Module):
    position = "absolute"

    def __init__(self, c: BertConfig):
        super().__init__()
        self.h, self.d = c.num_attention_heads, c.hidden_size // c.num_attention_heads
        self.query = nn.Linear(c.hidden_size, c.hidden_size)
        self.key = nn.Linear(c.hidden_size, c.hidden_size)
        self.value = nn.Linear(c.hidden_size, c.hidden_size)
        self.dropout = nn.Dropout(c.attention_probs_dropout_prob)
        self.position = getattr(c, "position_embedding_type", "absolute")  # (configurations from before there was a choice)
        if self.position == "relative_bias":
            self.max_distance = c.relative_attention_max_distance
            self.relative_bias = nn.Parameter(torch.zeros(c.relative_attention_num_buckets, self.h))
        elif self.position == "rotary":
            self.query_norm = nn.Parameter(torch.ones(self.d))
            self.key_norm = nn.Parameter(torch.ones(self.d))
            angle = torch.arange(c.max_position_embeddings, dtype=torch.float64)[:, None] * (
                c.rotary_base ** (-torch.arange(0, self.d, 2, dtype=torch.float64) / self.d))
            self.register_buffer("rotary_cos", angle.cos().float(), persistent=False)
            self.register_buffer("rotary_sin", angle.sin().float(), persistent=False)
        elif self.position != "absolute":
            raise ValueError(f"position_embedding_type must be 'absolute', 'relative_bias' or 'rotary', got {self.position!r}")

    def _project(self, x):
        """Queries, keys and values as [B, L, h, d], the first two rotated by position where the model does that."""
        B, L, _ = x.shape
        q, k, v = (p(x).view(B, L, self.h, self.d) for p in (self.query, self.key, self.value))
        if self.position == "rotary":
            from catch_b200.fusion import qk_norm_rotary

            q, k = qk_norm_rotary(q, k, self.query_norm, self.key_norm, self.rotary_cos, self.rotary_sin)
        return q, k, v

    def _biased_probs(self, scores, mask, scale):
        """Softmax of [B, h, L, L] scores, times ``scale``, with the relative position bias."""
        from catch_b200.fusion import relative_bias_softmax

        return relative_bias_softmax(scores, self.relative_bias, mask, scale=scale, max_distance=self.max_distance)

    def forward(self, x, mask=None):
        B, L, H = x.shape

        def split(t):  # [B, L, h, d] -> [B*h, L, d]
            return t.permute(0, 2, 1, 3).reshape(B * self.h, L, self.d)

        q, k, v = (split(t) for t in self._project(x))
        scores = torch.bmm(q, k.transpose(1, 2))
        if self.position == "relative_bias":
            probs = self._biased_probs(scores.view(B, self.h, L, L), mask, 1.0 / math.sqrt(self.d)).view(B * self.h, L, L)
        else:
            scores = scores * (1.0 / math.sqrt(self.d))
            if mask is not None:
                scores = scores.view(B, self.h, L, L) + mask
                scores = scores.view(B * self.h, L, L)
            probs = torch.softmax(scores, dim=-1)
        probs = self.dropout(probs)
        ctx = torch.bmm(probs, v).view(B, self.h, L, self.d).permute(0, 2, 1, 3).reshape(B, L, H)
        return ctx


class BertLayer(nn.Module):
    def __init__(self, c: BertConfig):
        super().__init__()
        self.attention = BertSelfAttention(c)
        self.attn_out = nn.Linear(c.hidden_size, c.hidden_size)
        self.attn_norm = nn.LayerNorm(c.hidden_size, eps=c.layer_norm_eps)
        self.intermediate = nn.Linear(c.hidden_size, c.intermediate_size)
        self.output = nn.Linear(c.intermediate_size, c.hidden_size)
        self.out_norm = nn.LayerNorm(c.hidden_size, eps=c.layer_norm_eps)
        self.dropout = nn.Dropout(c.hidden_dropout_prob)
        self.act = nn.GELU()

    def forward(self, x, mask=None):
        x = self.attn_norm(x + self.dropout(self.attn_out(self.attention(x, mask))))
        return self.out_norm(x + self.dropout(self.output(self.act(self.intermediate(x)))))


class FusedBertSelfAttention(BertSelfAttention):
    """Same parameters; the head split is a view and the two batched products read / write those views directly
    (``catch_b200.fusion.matmul_nd``), so no [batch * heads, seq, dim] copies are made in either direction."""

    def forward(self, x, mask=None):
        from catch_b200.fusion import matmul_nd

        if x.device.type != "blackwell" or not torch.is_autocast_enabled("blackwell"):
            return super().forward(x, mask)
        B, L, H = x.shape
        cd = torch.get_autocast_dtype("blackwell")

        def heads(t):  # [B, L, h, d] -> [B, h, L, d] view
            return t.to(cd).permute(0, 2, 1, 3)

        q, k, v = (heads(t) for t in self._project(x))
        scores = matmul_nd(q, k.transpose(-1, -2), 1.0 / math.sqrt(self.d))  # (scaled before they are rounded: the range of fp16)
        if self.position == "relative_bias":
            probs = self._biased_probs(scores, mask, 1.0)  # bias, mask and softmax in one kernel
        else:
            if mask is not None:
                scores = scores + mask.to(scores.dtype)
            with torch.autocast("blackwell", enabled=False):  # the softmax kernel computes in fp32 whatever the storage type
                probs = torch.softmax(scores, dim=-1)
        probs = self.dropout(probs)
        # the context is produced straight in [B, L, h, d] memory, seen as [B, h, L, d] by the product
        ctx = matmul_nd(probs, v, 1.0, (L * H, self.d, H, 1))
        return ctx.permute(0, 2, 1, 3).reshape(B, L, H)


class FusedBertLayer(BertLayer):
    """Same parameters; ``norm(x + dropout(h))`` runs as one fused kernel per direction."""

    def forward(self, x, mask=None):
        from catch_b200.fusion import dropout_add_layer_norm

        if x.device.type != "blackwell":
            return super().forward(x, mask)
        h = self.attn_out(self.attention(x, mask))
        x = dropout_add_layer_norm(h, x.to(h.dtype), self.attn_norm, self.dropout.p, self.training)
        h = self.output(self.act(self.intermediate(x)))
        return dropout_add_layer_norm(h, x.to(h.dtype), self.out_norm, self.dropout.p, self.training)


def fuse_bert(model: nn.Module) -> nn.Module:
    """Switch the layers of a BERT model to their fused forms and its linears to ``FusedLinear`` (in place; the
    parameters and the state dict are unchanged)."""
    from catch_b200.fusion import fuse_linear

    for m in model.modules():
        if type(m) is BertLayer:
            m.__class__ = FusedBertLayer
        elif type(m) is BertSelfAttention:
            m.__class__ = FusedBertSelfAttention
    return fuse_linear(model)


class BertForSequenceClassification(nn.Module):
    def __init__(self, config: BertConfig = None):
        super().__init__()
        c = self.config = config or BertConfig()
        self.embeddings = BertEmbeddings(c)
        self.layers = nn.ModuleList(BertLayer(c) for _ in range(c.num_hidden_layers))
        self.pooler = nn.Linear(c.hidden_size, c.hidden_size)
        self.dropout = nn.Dropout(c.hidden_dropout_prob)
        self.classifier = nn.Linear(c.hidden_size, c.num_labels)
        self.apply(self._init)

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, std=0.02)
        if isinstance(m, nn.Linear) and m.bias is not None:
            nn.init.zeros_(m.bias)

    def forward(self, input_ids, attention_mask=None, token_type_ids=None):
        mask = None
        if attention_mask is not None:
            mask = (1.0 - attention_mask[:, None, None, :].to(torch.float32)) * -10000.0
        x = self.embeddings(input_ids, token_type_ids)
        for layer in self.layers:
            x = layer(x, mask)
        pooled = torch.tanh(self.pooler(x[:, 0]))
        return self.classifier(self.dropout(pooled))
