"""Fine-tune LoRA adapters on a frozen NF4 model, everything on one GPU.

A small decoder (random weights, synthetic tokens) with NF4 projections: adapters on the attention
projections and the MLPs' down projections, the gate and up projections with their gating as one
operator, the frozen head under the chunked loss, and AdamW with 8-bit states, fp32 masters and
clipping, whose step reads the gradient norm on the GPU.

    python examples/finetune_adapters.py [--steps 30] [--bits 8]
"""

import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from stratum_amd import AdamW, NF4Linear, NF4LoRALinear, quantize_4bit  # noqa: E402
from stratum_amd.chunked_loss import chunked_linear_cross_entropy  # noqa: E402
from stratum_amd.mlp import NF4GatedMLP, quantize_mlp_  # noqa: E402


def frozen(out_features, in_features, rank=0):
    """A frozen random projection in NF4, with an adapter of that rank."""
    w = torch.randn(out_features, in_features, device="cuda", dtype=torch.bfloat16) * in_features ** -0.5
    packed, state = quantize_4bit(w)
    return NF4LoRALinear(packed, state, r=rank, lora_alpha=2.0 * rank) if rank else NF4Linear(packed, state)


class DenseMLP(nn.Module):
    def __init__(self, hidden, inter):
        super().__init__()
        self.gate_proj, self.up_proj = (nn.Linear(hidden, inter, bias=False) for _ in range(2))
        self.down_proj = nn.Linear(inter, hidden, bias=False)
        self.act_fn = nn.SiLU()


class Layer(nn.Module):
    def __init__(self, hidden, inter, heads, rank):
        super().__init__()
        self.heads = heads
        self.q, self.k, self.v, self.o = (frozen(hidden, hidden, rank) for _ in range(4))
        mlp = quantize_mlp_(DenseMLP(hidden, inter).to("cuda", torch.bfloat16).requires_grad_(False))
        mlp.down_proj = frozen(hidden, inter, rank)
        self.mlp = NF4GatedMLP(mlp)

    def forward(self, x):
        batch, length, hidden = x.shape
        y = F.rms_norm(x, (hidden,))
        q, k, v = (p(y).view(batch, length, self.heads, -1).transpose(1, 2) for p in (self.q, self.k, self.v))
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        x = x + self.o(y.transpose(1, 2).reshape(batch, length, hidden))
        return x + self.mlp(F.rms_norm(x, (hidden,)))


def train(steps=30, bits=8, hidden=512, inter=1408, layers=2, vocab=1000, batch=8, length=128, rank=16, seed=0):
    """Losses and gradient norms of every step (still on the GPU)."""
    torch.manual_seed(seed)
    embed = torch.randn(vocab, hidden, device="cuda", dtype=torch.bfloat16)
    model = nn.ModuleList(Layer(hidden, inter, 8, rank) for _ in range(layers))
    head = frozen(vocab // 8 * 8, hidden)
    adapters = [p for p in model.parameters() if p.requires_grad]
    optimizer = AdamW(adapters, lr=2e-3, weight_decay=0.0, state_bits=bits, master_weights=True, max_grad_norm=1.0)
    tokens = torch.randint(0, head.out_features, (batch, length + 1), device="cuda")
    losses, norms = [], []
    for _ in range(steps):
        x = embed[tokens[:, :-1]]
        for layer in model:
            x = layer(x)
        loss = chunked_linear_cross_entropy(F.rms_norm(x, (hidden,)), head, tokens[:, 1:])
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        norms.append(optimizer.grad_norm[0])
    return torch.stack(losses), torch.stack(norms)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--bits", type=int, default=8, choices=(8, 32))
    a = ap.parse_args()
    losses, norms = train(a.steps, a.bits)
    for i, (loss, norm) in enumerate(zip(losses.tolist(), norms.tolist())):
        print(f"step {i:3d}  loss {loss:.4f}  gradient norm {norm:.4f}")
