"""A small language model of selective scan blocks: a student that learns from a teacher's top logits, then answers.

Each block is layer norm -> projection -> short causal filter -> selective
scan -> gate -> projection, added to its input; a layer norm and the transposed
embedding give the logits.  The script trains such a model for a few steps with
the distillation loss, reads prompts of unequal lengths in one call and goes on
token by token from the states that they leave.

    python bayes-ssm_amd/examples/selective_lm.py --device cuda --dtype bfloat16
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch import Tensor

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from bayes_ssm.conv import causal_conv
from bayes_ssm.distill import distillation_loss
from bayes_ssm.norm import LayerNorm
from bayes_ssm.selective import selective_scan, selective_step

State = tuple[Tensor, Tensor]  # the filter's last inputs, the scan's state


class SelectiveBlock(nn.Module):
    """``x + out(scan(filter(in(norm(x)))) * silu(gate))``."""

    def __init__(self, width: int, heads: int, values: int, n: int, groups: int = 1, taps: int = 4):
        super().__init__()
        self.heads, self.values, self.n, self.groups = heads, values, n, groups
        inner, channels = heads * values, heads * values + 2 * groups * n
        self.norm = LayerNorm(width)
        self.inp = nn.Linear(width, inner + channels + heads, bias=False)  # gate | filter's channels | steps
        self.out = nn.Linear(inner, width, bias=False)
        self.conv_weight = nn.Parameter(torch.randn(channels, taps) / taps**0.5)
        self.conv_bias = nn.Parameter(torch.zeros(channels))
        self.log_rate = nn.Parameter(torch.linspace(0.0, 2.0, heads))
        self.skip = nn.Parameter(torch.ones(heads))
        self.dt_bias = nn.Parameter(torch.linspace(-4.0, -1.0, heads))

    def _parts(self, x: Tensor) -> tuple[Tensor, Tensor, Tensor]:
        inner = self.heads * self.values
        row = self.inp(self.norm(x))
        return row[..., :inner], row[..., inner:-self.heads], row[..., -self.heads:]

    def forward(self, x: Tensor, lengths: Optional[Tensor] = None) -> tuple[Tensor, State]:
        b, t = x.shape[:2]
        inner, gn = self.heads * self.values, self.groups * self.n
        gate, channels, dt = self._parts(x)
        row, conv_state = causal_conv(channels, self.conv_weight, self.conv_bias, activation="silu", lengths=lengths)
        v, B, C = row[..., :inner], row[..., inner:inner + gn], row[..., inner + gn:]
        y, state = selective_scan(
            v.unflatten(-1, (self.heads, self.values)), dt, -torch.exp(self.log_rate),
            B.unflatten(-1, (self.groups, self.n)), C.unflatten(-1, (self.groups, self.n)), D=self.skip,
            dt_bias=self.dt_bias, lengths=lengths)
        return x + self.out(y.reshape(b, t, inner) * F.silu(gate)), (conv_state, state)

    def step(self, x: Tensor, state: State) -> tuple[Tensor, State]:
        gate, channels, dt = self._parts(x)
        y, conv_state, scan_state = selective_step(
            channels, dt, *state, self.conv_weight, -torch.exp(self.log_rate), groups=self.groups,
            conv_bias=self.conv_bias, D=self.skip, dt_bias=self.dt_bias,
            out_states=(torch.empty_like(state[0]), state[1]))  # the scan's state in place
        return x + self.out(y.flatten(1) * F.silu(gate)), (conv_state, scan_state)


class SelectiveLM(nn.Module):
    def __init__(self, vocabulary: int, width: int = 128, blocks: int = 2, heads: int = 4, values: int = 32, n: int = 32):
        super().__init__()
        self.embed = nn.Embedding(vocabulary, width)
        nn.init.normal_(self.embed.weight, std=width**-0.5)
        self.blocks = nn.ModuleList(SelectiveBlock(width, heads, values, n) for _ in range(blocks))
        self.norm = LayerNorm(width)

    def _logits(self, x: Tensor) -> Tensor:
        return F.linear(self.norm(x), self.embed.weight)

    def forward(self, tokens: Tensor, lengths: Optional[Tensor] = None) -> tuple[Tensor, list[State]]:
        """Logits [batch, time, vocabulary] and the states behind each row's last token."""
        x, states = self.embed(tokens), []
        for block in self.blocks:
            x, state = block(x, lengths)
            states.append(state)
        return self._logits(x), states

    @torch.no_grad()
    def step(self, tokens: Tensor, states: list[State]) -> tuple[Tensor, list[State]]:
        """Logits [batch, vocabulary] after one more token a row."""
        x, after = self.embed(tokens), []
        for block, state in zip(self.blocks, states):
            x, state = block.step(x, state)
            after.append(state)
        return self._logits(x), after


def train_step(model: SelectiveLM, optimizer: torch.optim.Optimizer, tokens: Tensor, teacher_logits: Tensor,
               teacher_index: Tensor, temperature: float = 2.0) -> Tensor:
    """One distillation step; positions whose teacher_index is -1 throughout do not count."""
    logits, _ = model(tokens)
    loss = distillation_loss(logits, teacher_logits, teacher_index, temperature=temperature)
    optimizer.zero_grad(set_to_none=True)
    loss.backward()
    optimizer.step()
    return loss.detach()


@torch.no_grad()
def generate(model: SelectiveLM, prompts: Tensor, lengths: Tensor, count: int) -> Tensor:
    """``count`` greedy tokens behind each of the prompts [batch, time], whose rows have ``lengths`` (at least 1)."""
    logits, states = model(prompts, lengths)
    last = logits[torch.arange(len(lengths), device=prompts.device), lengths - 1]
    out = []
    for _ in range(count):
        out.append(last.argmax(-1))
        last, states = model.step(out[-1], states)
    return torch.stack(out, 1)


def teach(tokens: Tensor, vocabulary: int, entries: int = 8) -> tuple[Tensor, Tensor]:
    """A made-up teacher: the next token is the last one times 5 plus 1, the entries around it fall off; a row's first
    tokens are prompt and have none."""
    at = torch.arange(entries, device=tokens.device)
    index = (tokens[..., None] * 5 + 1 + at) % vocabulary
    index[:, :2] = -1
    return (-0.7 * at).expand(index.shape), index


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    parser.add_argument("--dtype", default="float32", choices=("float32", "bfloat16"))
    parser.add_argument("--steps", type=int, default=60)
    args = parser.parse_args()
    torch.manual_seed(0)
    vocabulary = 97
    model = SelectiveLM(vocabulary).to(args.device, getattr(torch, args.dtype))
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3)
    for k in range(args.steps):
        tokens = torch.randint(0, vocabulary, (8, 96), device=args.device)
        loss = train_step(model, optimizer, tokens, *teach(tokens, vocabulary))
        if k % 20 == 0 or k == args.steps - 1:
            print(f"step {k}: loss {loss.item():.4f}", flush=True)
    prompts = torch.randint(0, vocabulary, (3, 40), device=args.device)
    lengths = torch.tensor([40, 17, 1], device=args.device)
    print("answers:", generate(model, prompts, lengths, 6).tolist())


if __name__ == "__main__":
    main()
