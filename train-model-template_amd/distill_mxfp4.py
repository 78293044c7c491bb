"""A small example that runs the 4-bit operators together as a program would: a language model's gated MLPs are quantized to
MXFP4 (mxfp4.enable_mxfp4), LoRA adapters on top of them learn what a finetuned model of the same base knows from its top
logits (distill.topk_kl_rows), and the student then answers one token at a time.

    python train-model-template_amd/distill_mxfp4.py --steps 200

Random weights and tokens: a token and the one before it are embedded, pass gated MLPs with residuals and norms, and a head
gives logits over the vocabulary.
"""
import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import distill  # noqa: E402
import mxfp4  # noqa: E402
import workloads  # noqa: E402


class Model(nn.Module):
    """layers of workloads.SwiGLUMLP (LoRA on gate, up and down) between embeddings and a head.  learned: the adapters' B is
    random (a finetuned model), else zero (the start of training); the rest depends on the seed alone."""

    def __init__(self, layers, d, ffn, vocab, rank, learned, seed=0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        r = lambda *s, std: torch.randn(*s, generator=g) * std  # noqa: E731
        self.embed = nn.Parameter(r(2, vocab, d, std=1.0).to(torch.bfloat16), requires_grad=False)
        self.head = nn.Parameter(r(vocab, d, std=3.0 * d ** -0.5).to(torch.bfloat16), requires_grad=False)
        mlps = []
        for _ in range(layers):
            inp = dict(K=d, N=ffn, Wg=r(ffn, d, std=2 * d ** -0.5), Wu=r(ffn, d, std=2 * d ** -0.5),
                       Wd=r(d, ffn, std=2 * ffn ** -0.5))
            for n, (o, i) in dict(g=(ffn, d), u=(ffn, d), d=(d, ffn)).items():
                inp["A" + n], inp["B" + n] = r(rank, i, std=i ** -0.5), r(o, rank, std=0.3 if learned else 0.0)
            mlps.append(workloads.SwiGLUMLP(inp, rank))
            for n in ("gate_proj", "up_proj", "down_proj"):
                getattr(mlps[-1], n).base_layer.to(torch.bfloat16)
        self.model = workloads.MLPStack(mlps).model

    def forward(self, tokens, before):
        """Logits [T, vocab] of the tokens that follow `tokens`, `before` the ones in front of them."""
        norm = lambda t: nn.functional.rms_norm(t, t.shape[-1:]).to(torch.bfloat16)  # noqa: E731
        with torch.autocast(self.head.device.type, torch.bfloat16):  # the adapters are fp32
            x = self.embed[0][tokens] + self.embed[1][before]
            for layer in self.model.layers:
                x = x + layer.mlp(norm(x))
            return norm(x) @ self.head.t()

    @torch.no_grad()
    def answer(self, first, n):
        """n tokens after `first` (a list of two), the likeliest each time: the single-token forms."""
        out = list(first)
        dev = self.head.device
        for _ in range(n):
            z = self(torch.tensor([out[-1]], device=dev), torch.tensor([out[-2]], device=dev))
            out.append(int(z[0].argmax()))
        return out


def run(steps=200, tokens=2048, layers=2, d=512, ffn=1536, vocab=8192, rank=16, k=32, lr=2e-3, act="e4m3", device="cuda",
        log=print):
    """The example; returns its figures."""
    teacher = Model(layers, d, ffn, vocab, rank, True).to(device)
    student = Model(layers, d, ffn, vocab, rank, False).to(device)
    n = mxfp4.enable_mxfp4(student, act=act)
    adapters = [p for p in student.parameters() if p.requires_grad]
    opt = torch.optim.AdamW(adapters, lr=lr, weight_decay=0.0)
    gen = torch.Generator().manual_seed(1)

    def batch():
        t = torch.randint(0, vocab, (tokens + 1,), generator=gen).to(device)
        with torch.no_grad():
            z = teacher(t[1:], t[:-1]).float()
        top, idx = z.topk(k, dim=1)
        return t[1:], t[:-1], idx.to(torch.int32), top, torch.logsumexp(z, 1)

    held = batch()

    def evaluate():
        with torch.no_grad():
            return distill.topk_kl(student(*held[:2]), *held[2:4], teacher_lse=held[4]).mean().item()

    start = evaluate()
    weight = torch.full((tokens,), 1.0 / tokens, device=device)
    for step in range(steps):
        now, before, idx, top, lse = batch()
        z = student(now, before)
        loss, grad = distill.topk_kl_rows(z, idx, top, weight, teacher_lse=lse)
        opt.zero_grad(set_to_none=True)
        z.backward(grad)
        opt.step()
        if step % 40 == 0:
            log(f"step {step}: divergence {loss.mean().item():.4f}")
    end = evaluate()
    mine, theirs = student.answer([3, 5], 8), teacher.answer([3, 5], 8)
    log(f"{n} linears in MXFP4; divergence from the teacher on held-out tokens {start:.4f} -> {end:.4f}")
    log(f"student {mine}\nteacher {theirs}")
    return dict(start=start, end=end, linears=n, student=student, teacher=teacher, held=held)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--act", choices=("e4m3", "e2m1"), default="e4m3")
    a = ap.parse_args()
    run(a.steps, a.tokens, act=a.act)
