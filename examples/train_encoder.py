"""A late-interaction model trained from token ids to MaxSim scores on one GPU.

A small pre-norm transformer encoder from the library's operators (layer norm
with the residual sum, attention over padded rows, gated feed-forward block), the
projection head fused into the scoring (``maxsim_from_hidden``), and the
in-batch contrastive loss. Data are synthetic: some of a query's tokens are drawn from
its own passage.

    python examples/train_encoder.py [steps]
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

_PKG = str(Path(__file__).resolve().parents[1] / "late-interaction-kernels_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

from late_interaction_kernels.encoder import attention, gated_ffn, layer_norm  # noqa: E402
from late_interaction_kernels.fused_head import maxsim_from_hidden  # noqa: E402


class EncoderLayer(nn.Module):
    """``s`` is the residual stream; ``x`` what the layer before adds to it."""

    def __init__(self, d: int, heads: int, kv_heads: int, hidden: int, window: int | None = None):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim, self.window = heads, kv_heads, d // heads, window

        def weight(rows, cols):
            return nn.Parameter(torch.randn(rows, cols) * cols**-0.5)

        self.norm_att = nn.Parameter(torch.ones(d))
        self.norm_ffn = nn.Parameter(torch.ones(d))
        self.w_qkv = weight((heads + 2 * kv_heads) * self.head_dim, d)
        self.w_att = weight(d, heads * self.head_dim)
        self.w_in = weight(2 * hidden, d)
        self.w_out = weight(d, hidden)

    def forward(self, x: torch.Tensor, s: torch.Tensor, mask: torch.Tensor):
        n, length, d = x.shape
        y, s = layer_norm(x, self.norm_att, None, s)
        qkv = F.linear(y, self.w_qkv).view(n, length, self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=2)
        a = attention(q, k, v, mask, mask, window=self.window)
        y, s = layer_norm(F.linear(a.reshape(n, length, -1), self.w_att), self.norm_ffn, None, s)
        return gated_ffn(y, self.w_in, self.w_out), s


class Encoder(nn.Module):
    def __init__(self, vocab=2048, d=256, layers=2, heads=4, kv_heads=2, hidden=384, d_out=128):
        super().__init__()
        self.embed = nn.Parameter(torch.randn(vocab, d))
        self.layers = nn.ModuleList(
            EncoderLayer(d, heads, kv_heads, hidden, window=None if i % 2 else 16) for i in range(layers))
        self.norm = nn.Parameter(torch.ones(d))
        self.head = nn.Parameter(torch.randn(d_out, d) * d**-0.5)

    def hidden_states(self, ids: torch.Tensor, mask: torch.Tensor) -> torch.Tensor:
        x = F.embedding(ids, self.embed)
        s = torch.zeros_like(x)
        for layer in self.layers:
            x, s = layer(x, s, mask)
        return layer_norm(x, self.norm, None, s)[0]

    def scores(self, q_ids, q_mask, d_ids, d_mask) -> torch.Tensor:
        q = F.normalize(F.linear(self.hidden_states(q_ids, q_mask), self.head).float(), dim=-1)
        q = (q * q_mask[..., None]).to(self.head.dtype)
        return maxsim_from_hidden(q, self.hidden_states(d_ids, d_mask), self.head, None, d_mask)


def batch(n: int, lq: int, ld: int, vocab: int, seed: int):
    """``n`` passages of up to ``ld`` tokens, and for each a query of up to ``lq``: three in ten are the passage's."""
    g = torch.Generator().manual_seed(seed)
    d_len = torch.randint(ld // 4, ld + 1, (n,), generator=g)
    q_len = torch.randint(lq // 2, lq + 1, (n,), generator=g)
    d_ids = torch.randint(vocab, (n, ld), generator=g)
    at = (torch.rand(n, lq, generator=g) * d_len[:, None]).long()
    q_ids = torch.where(torch.rand(n, lq, generator=g) < 0.3, d_ids.gather(1, at),
                        torch.randint(vocab, (n, lq), generator=g))
    masks = torch.arange(lq)[None] < q_len[:, None], torch.arange(ld)[None] < d_len[:, None]
    return tuple(t.cuda() for t in (q_ids, masks[0], d_ids, masks[1]))


def train(steps: int = 40, n: int = 32, seed: int = 0) -> list[float]:
    """Trains on four batches in turn; returns the losses."""
    torch.manual_seed(seed)
    model = Encoder().cuda().to(torch.bfloat16)
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3)
    target = torch.arange(n, device="cuda")
    losses = []
    for step in range(steps):
        scores = model.scores(*batch(n, 16, 96, 2048, step % 4))
        loss = F.cross_entropy(scores, target)
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    got = train(int(sys.argv[1]) if len(sys.argv) > 1 else 40)
    for i in range(0, len(got), max(1, len(got) // 8)):
        print(f"step {i}: loss {got[i]:.3f}")
    print(f"last: {got[-1]:.3f}")
