"""An expert layer whose routing is an exact assignment.

A router scores every token against every expert.  Each expert offers the same
number of slots, and the auction solver assigns tokens to slots so that the total
score is best, so every expert gets the same load without a balancing loss.  The
tokens then go through the expert operators: sorted by expert, two grouped
products, and back, weighted by the gate of the expert they were given.

    python examples/balanced_experts.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import efficient_linear_assignment_b200 as ela  # noqa: E402


class BalancedExperts(torch.nn.Module):
    def __init__(self, hidden, width, experts, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.experts = experts

        def weights(*shape):
            return torch.nn.Parameter(torch.randn(*shape, device=device, dtype=torch.float32).mul_(shape[-1] ** -0.5).to(dtype))

        self.router = torch.nn.Parameter(torch.randn(experts, hidden, device=device) * hidden ** -0.5)
        self.w1, self.b1 = weights(experts, width, hidden), torch.nn.Parameter(torch.zeros(experts, width, device=device, dtype=dtype))
        self.w2, self.b2 = weights(experts, hidden, width), torch.nn.Parameter(torch.zeros(experts, hidden, device=device, dtype=dtype))

    def assign(self, score, max_iter=1000):
        """(T, E) scores -> expert of each token, -1 for a token the auction left out.
        Slot s belongs to expert s // slots, and costs a token minus its score there."""
        tokens, experts = score.shape
        slots = -(-tokens // experts)
        slots += -slots % 2
        cost = (-score.detach()).repeat_interleave(slots, dim=1).unsqueeze(0)
        slot, _ = ela.AuctionB200(epsilon=[0.1, 0.02], max_iter=max_iter).solve(cost)
        return torch.where(slot[0] >= 0, slot[0] // slots, slot[0])

    def forward(self, x, expert=None):
        score = x.float() @ self.router.t()
        if expert is None:
            expert = self.assign(score)
        plan = ela.expert_plan(expert, self.experts)
        gate = torch.sigmoid(score.gather(1, expert.clamp(min=0).unsqueeze(1)))
        rows = ela.expert_dispatch(x, plan)
        h = ela.expert_linear(rows, self.w1, self.b1, activation="gelu", offsets=plan.offsets)
        h = ela.expert_linear(h, self.w2, self.b2, offsets=plan.offsets)
        return x + ela.expert_combine(h, plan, gate)


def train(steps=100, tokens=4096, hidden=512, width=2048, experts=16, verbose=True):
    """Fits a random function of the token; returns the losses."""
    torch.manual_seed(0)
    layer = BalancedExperts(hidden, width, experts)
    target = torch.randn(hidden, hidden, device="cuda") * hidden ** -0.5
    opt = torch.optim.AdamW(layer.parameters(), lr=2e-3)
    losses = []
    for step in range(steps):
        x = torch.randn(tokens, hidden, device="cuda").to(torch.bfloat16)
        out = layer(x)
        loss = (out.float() - torch.tanh(x.float() @ target)).square().mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.item())
        if verbose and step % 20 == 0:
            print(f"step {step:4d}  loss {losses[-1]:.4f}")
    ela.expert_check()
    return losses


def generate(steps=100, tokens=8, hidden=1024, width=4096, experts=16, verbose=True):
    """Single steps of a few tokens: the whole layer after the routing in one CUDA graph."""
    torch.manual_seed(1)
    layer = BalancedExperts(hidden, width, experts)
    x = torch.randn(tokens, hidden, device="cuda").to(torch.bfloat16)
    expert = torch.zeros(tokens, dtype=torch.int64, device="cuda")
    with torch.no_grad():
        layer(x, expert)  # first calls outside the capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(x, expert)
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(steps):
            expert.copy_((x.float() @ layer.router.t()).argmax(1))  # a few tokens go where they like
            graph.replay()
            x.copy_(y / y.float().square().mean(1, keepdim=True).sqrt().to(y.dtype))
        end.record()
        torch.cuda.synchronize()
    ela.expert_check()
    if verbose:
        print(f"{begin.elapsed_time(end) / steps * 1000:.1f} us a step of {tokens} tokens")
    return bool(torch.isfinite(y).all())


if __name__ == "__main__":
    train()
    generate()
