"""Train a small language model of gated feed-forward blocks and score text with its head in 8 bits: came_amd's embedding, norm with
the residual's addition, feed-forward block, token log probabilities and optimizer step as one loop, then the 8-bit norm and
product.

    python examples/train_language_model.py --optimizer adamw8bit --steps 200

The text is drawn from a random Markov chain, so that a token is all that its follower depends on.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import came_amd  # noqa: E402

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
LRS = {"adamw": 3e-3, "adamw8bit": 3e-3, "came8bit": 2e-4}  # CAME's steps are larger at the same rate
PADDING = 0  # the token that ends a shorter sequence


class Model(torch.nn.Module):
    """embedding, blocks of h + gated_ffn(norm(h)), norm, head; each norm adds what the block before it has made."""

    def __init__(self, vocab: int, dim: int, hidden: int, layers: int, dtype: torch.dtype, gen: torch.Generator):
        super().__init__()

        def weight(*shape):
            return torch.nn.Parameter((torch.randn(*shape, generator=gen) * shape[-1] ** -0.5).to(dtype).cuda())

        self.table, self.head = weight(vocab, dim), weight(vocab, dim)
        self.blocks = torch.nn.ModuleList(torch.nn.ParameterDict({
            "gate": weight(hidden, dim), "up": weight(hidden, dim), "down": weight(dim, hidden)}) for _ in range(layers))
        self.norms = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(dim, dtype=dtype, device="cuda")) for _ in range(layers + 1))

    def stream(self, tokens: torch.Tensor):
        """What the last norm takes: the last block's result and the residual stream."""
        x, h = came_amd.embedding(tokens, self.table, scale=self.table.shape[1] ** 0.5, padding_idx=PADDING), None
        for norm, w in zip(self.norms, self.blocks):
            if h is None:
                y, h = came_amd.rms_norm(x, norm), x
            else:
                y, h = came_amd.rms_norm(x, norm, residual=h)
            x = came_amd.gated_ffn(y, w["gate"], w["up"], w["down"])
        return x, h

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        x, h = self.stream(tokens)
        return came_amd.rms_norm(x, self.norms[-1], residual=h)[0] @ self.head.t()


def loss_of(logits: torch.Tensor, followers: torch.Tensor, bonus: float = 0.0) -> torch.Tensor:
    """Mean negative log probability of the followers, those that are padding left out, less a bonus for entropy."""
    given = followers != PADDING
    r = came_amd.token_log_probs(logits, torch.where(given, followers, -100))
    return -r.log_probs.sum() / given.sum() - bonus * r.entropy.mean()


class Scorer:
    """The model for serving, its head in 8 bits: log probabilities of a text and the alternatives at every place."""

    def __init__(self, model: Model):
        self.model = model
        self.head, self.scale = came_amd.quantize_rows(model.head.detach())

    @torch.no_grad()
    def __call__(self, tokens: torch.Tensor, top: int = 5) -> came_amd.TokenLogProbs:
        x, h = self.model.stream(tokens[..., :-1])
        q, s, _ = came_amd.rms_norm_int8(x, self.model.norms[-1], residual=h)
        logits = came_amd.int8_linear(q, s, self.head, self.scale, dtype=torch.float32)
        return came_amd.token_log_probs(logits, tokens[..., 1:], top=top)


def text(chain: torch.Tensor, batch: int, length: int, gen: torch.Generator) -> torch.Tensor:
    """Sequences of the chain, some of them shorter and padded."""
    t = torch.randint(1, chain.shape[0], (batch, 1), generator=gen)
    for _ in range(length):
        t = torch.cat((t, torch.multinomial(chain[t[:, -1]], 1, generator=gen)), 1)
    ends = torch.randint(length // 2, length + 2, (batch, 1), generator=gen)
    return torch.where(torch.arange(length + 1) < ends, t, PADDING)


def optimizer(name: str, params, lr: float):
    if name == "adamw":
        return came_amd.AdamW(params, lr=lr, max_grad_norm=1.0)
    if name == "adamw8bit":
        return came_amd.AdamW8bit(params, lr=lr, max_grad_norm=1.0)
    return came_amd.CAME8bit(params, lr=lr, weight_decay=1e-2)


def train(steps: int = 200, vocab: int = 1000, dim: int = 256, hidden: int = 704, layers: int = 2, batch: int = 16, length: int = 64,
          name: str = "adamw8bit", dtype: str = "bf16", lr: float | None = None, log=print):
    """The trained model, the losses of every tenth step and the last, and a text that it has not seen."""
    gen = torch.Generator().manual_seed(0)
    chain = torch.exp(3 * torch.randn(vocab, vocab, generator=gen))
    chain[:, PADDING] = 0
    model = Model(vocab, dim, hidden, layers, DTYPES[dtype], gen)
    params = list(model.parameters())
    opt = optimizer(name, params, lr or LRS[name])
    losses = []
    for step in range(steps):
        t = text(chain, batch, length, gen).cuda()
        loss = loss_of(model(t[:, :-1]), t[:, 1:], bonus=1e-3)
        loss.backward()
        if not hasattr(opt, "max_grad_norm"):  # CAME clips each update by itself; the gradients' norm is clipped here
            came_amd.clip_grad_norm_(params, 1.0)
        opt.step()
        opt.zero_grad()
        if step % 10 == 0 or step == steps - 1:
            losses.append(float(loss.detach()))
            log(f"step {step:4d}  loss {losses[-1]:.4f}")
    return model, losses, text(chain, 4, length, gen).cuda()


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--optimizer", choices=sorted(LRS), default="adamw8bit")
    ap.add_argument("--dtype", choices=sorted(DTYPES), default="bf16")
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--lr", type=float)
    a = ap.parse_args()
    model, _, unseen = train(a.steps, name=a.optimizer, dtype=a.dtype, lr=a.lr)
    r = Scorer(model)(unseen)
    given = unseen[:, 1:] != PADDING
    print(f"unseen text, 8-bit head: {-r.log_probs[given].mean():.4f} a token, entropy {r.entropy[given].mean():.4f}; of the first, "
          f"{unseen[0, 1:6].tolist()} among {r.top_tokens[0, :5].tolist()}")


if __name__ == "__main__":
    main()
