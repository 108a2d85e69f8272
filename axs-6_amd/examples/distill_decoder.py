"""A quantized decoder trained from its full-precision teacher, then answering
from the 8-bit cache: the library's decoder operators together.

    python axs-6_amd/examples/distill_decoder.py [--steps 300] [--tokens 48]

1. A small float32 decoder (the teacher) learns sequences that count up in
   strides through a vocabulary.
2. The student has the same shape with every linear and embedding quantized to
   NF5, rotary positions and grouped heads; it never sees the data's labels, only
   the teacher's 16 top logits of each token (``axs_distillation_loss_unified``).
3. The student continues a prompt, token by token, from the 8-bit cache
   (``AXSCausalSelfAttentionUnified.decode``), then with four beams that share
   the prompt's cache (``axs_beam_search_unified``).
"""
from __future__ import annotations

import argparse
import os
import sys
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import axs.unified as axu  # noqa: E402


@dataclass
class Config:
    vocab: int = 256
    context: int = 128
    width: int = 256
    heads: int = 4
    kv_heads: int = 2
    layers: int = 2
    batch: int = 32
    lr: float = 1e-3
    top: int = 16
    temperature: float = 1.5


class Attention(nn.Module):
    """The teacher's: the student's operators around full-precision projections."""

    def __init__(self, c: Config) -> None:
        super().__init__()
        self.hd = c.width // c.heads
        self.q = nn.Linear(c.width, c.width)
        self.kv = nn.Linear(c.width, 2 * c.kv_heads * self.hd)
        self.o = nn.Linear(c.width, c.width)

    def forward(self, x: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
        q = self.q(x).unflatten(-1, (-1, self.hd))
        k, v = self.kv(x).unflatten(-1, (-1, self.hd)).chunk(2, dim=2)
        q, k = axu.axs_rotary_unified(q, k, table)
        return self.o(axu.axs_attention_unified(q, k, v, causal=True).flatten(2))


class Block(nn.Module):
    def __init__(self, c: Config, quantized: bool) -> None:
        super().__init__()
        norm = axu.AXSLayerNormUnified if quantized else nn.LayerNorm
        linear = axu.AXSLinearUnified if quantized else nn.Linear
        self.n1, self.n2 = norm(c.width), norm(c.width)
        self.attn = axu.AXSCausalSelfAttentionUnified(c.width, c.heads, c.kv_heads) if quantized else Attention(c)
        self.up, self.down = linear(c.width, 4 * c.width), linear(4 * c.width, c.width)

    def ffn(self, x: torch.Tensor) -> torch.Tensor:
        return x + self.down(F.gelu(self.up(self.n2(x))))

    def forward(self, x: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
        return self.ffn(x + self.attn(self.n1(x), table))

    def decode(self, x: torch.Tensor, table: torch.Tensor, cache: axu.AXSKVCacheUnified, starts: torch.Tensor, *prefix) -> torch.Tensor:
        return self.ffn(x + self.attn.decode(self.n1(x), table, cache, starts, *prefix))


class Decoder(nn.Module):
    def __init__(self, c: Config, quantized: bool) -> None:
        super().__init__()
        self.c = c
        self.embed = (axu.AXSEmbeddingUnified if quantized else nn.Embedding)(c.vocab, c.width)
        self.blocks = nn.ModuleList(Block(c, quantized) for _ in range(c.layers))
        self.norm = (axu.AXSLayerNormUnified if quantized else nn.LayerNorm)(c.width)
        self.head = (axu.AXSLinearUnified if quantized else nn.Linear)(c.width, c.vocab)
        self.register_buffer("table", axu.rotary_table(c.width // c.heads, 2 * c.context), persistent=False)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        x = self.embed(tokens)
        for b in self.blocks:
            x = b(x, self.table)
        return self.head(self.norm(x))

    @torch.no_grad()
    def logits_from_cache(self, tokens: torch.Tensor, caches: list, starts: torch.Tensor, prefixes: list | None = None,
                          lengths: torch.Tensor | None = None) -> torch.Tensor:
        """Logits of ``tokens`` (B, T), which follow the ``starts[b]`` tokens that the caches hold, and those before
        them of the shared prefixes, if any."""
        x = self.embed(tokens)
        for i, (b, cache) in enumerate(zip(self.blocks, caches)):
            x = b.decode(x, self.table, cache, starts, *(() if prefixes is None else (prefixes[i], lengths)))
        return self.head(self.norm(x))

    @torch.no_grad()
    def generate(self, prompt: torch.Tensor, count: int) -> torch.Tensor:
        """``prompt`` (B, T) and ``count`` more tokens, the likeliest each."""
        B, T = prompt.shape
        caches = [b.attn.new_cache(B, T + count, device=prompt.device) for b in self.blocks]
        starts = torch.zeros(B, dtype=torch.int64, device=prompt.device)
        out, new = [prompt], prompt
        for _ in range(count):
            logits = self.logits_from_cache(new, caches, starts)
            starts = starts + new.shape[1]
            new = logits[:, -1:].argmax(-1)
            out.append(new)
        return torch.cat(out, 1)

    @torch.no_grad()
    def generate_beams(self, prompt: torch.Tensor, count: int, beams: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The ``beams`` likeliest continuations found of each ``prompt`` (B, T) by ``count`` tokens: their log
        probabilities (B, beams) and the whole sequences (B, beams, T + count).  A prompt is cached once for all of
        its beams, which cache their own tokens alone."""
        B, T = prompt.shape
        prompts = [b.attn.new_cache(B, T, device=prompt.device) for b in self.blocks]
        caches = [b.attn.new_cache(B * beams, count, device=prompt.device) for b in self.blocks]
        lengths = torch.full((B,), T, dtype=torch.int64, device=prompt.device)
        logits = self.logits_from_cache(prompt, prompts, torch.zeros_like(lengths))[:, -1]
        scores, tokens = axu.axs_beam_search_unified(
            lambda new, starts: self.logits_from_cache(new, caches, starts, prompts, lengths), logits, caches, beams, count)
        return scores, torch.cat([prompt[:, None].expand(-1, beams, -1), tokens], -1)


def sequences(c: Config, g: torch.Generator, device: str) -> torch.Tensor:
    """(batch, context + 1): start + stride * position, modulo the vocabulary."""
    start = torch.randint(0, c.vocab, (c.batch, 1), generator=g)
    stride = torch.randint(1, 8, (c.batch, 1), generator=g)
    return ((start + stride * torch.arange(c.context + 1)) % c.vocab).to(device)


def train_teacher(c: Config, steps: int, device: str = "cuda") -> Decoder:
    torch.manual_seed(0)
    teacher, g = Decoder(c, False).to(device), torch.Generator().manual_seed(1)
    opt = torch.optim.AdamW(teacher.parameters(), lr=c.lr)
    for _ in range(steps):
        t = sequences(c, g, device)
        opt.zero_grad()
        F.cross_entropy(teacher(t[:, :-1]).flatten(0, 1), t[:, 1:].flatten()).backward()
        opt.step()
    return teacher


def distill(c: Config, teacher: Decoder, steps: int, device: str = "cuda") -> tuple[Decoder, list[float]]:
    torch.manual_seed(2)
    student, g = Decoder(c, True).to(device), torch.Generator().manual_seed(3)
    opt = torch.optim.AdamW(student.parameters(), lr=c.lr)
    losses = []
    for _ in range(steps):
        t = sequences(c, g, device)
        with torch.no_grad():
            values, classes = teacher(t[:, :-1]).topk(c.top, -1)
        opt.zero_grad()
        loss = axu.axs_distillation_loss_unified(student(t[:, :-1]), values, classes, c.temperature)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return student, torch.stack(losses).tolist()


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--tokens", type=int, default=48)
    a = ap.parse_args()
    c = Config()
    teacher = train_teacher(c, a.steps)
    student, losses = distill(c, teacher, a.steps)
    print(f"distillation loss {losses[0]:.3f} -> {losses[-1]:.3f} in {a.steps} steps")
    want = sequences(c, torch.Generator().manual_seed(4), "cuda")[:, :16 + a.tokens]
    got = student.generate(want[:, :16], a.tokens)
    share = float((got[:, 16:] == want[:, 16:]).float().mean())
    print(f"{a.tokens} tokens from the 8-bit cache after 16: {100 * share:.0f}% as the sequences go on")
    scores, got = student.generate_beams(want[:, :16], a.tokens, 4)
    share = float((got[:, 0, 16:] == want[:, 16:]).float().mean())
    print(f"the best of 4 beams: {100 * share:.0f}%, log probability {float(scores[:, 0].mean()):.2f}")


if __name__ == "__main__":
    main()
