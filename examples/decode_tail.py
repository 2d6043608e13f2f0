"""Greedy decoding through the operators behind a decode step's attention.

Each step takes one token a request: an embedding row, a mixture-of-experts
layer (router, routed and shared experts), a 4-bit vocabulary projection, then
biases, penalties and a mask of allowed tokens on the logits, and the largest
one is appended to the request's history.  Attention is left out, weights are
random; what stays is the chain of calls as a serving loop makes it, captured
once in a CUDA graph and replayed per step.

    python examples/decode_tail.py --requests 4 --steps 32 --weights w4
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-ernie_b200"))

from vllm_ernie_b200 import ops  # noqa: E402


def random_experts(kind: str, lead: tuple, hidden: int, inner: int) -> ops.MoEWeights:
    """Random gated MLPs ``[*lead]`` in one of the three weight formats."""
    w13 = torch.randn((*lead, 2 * inner, hidden), device="cuda") / hidden ** 0.5
    w2 = torch.randn((*lead, hidden, inner), device="cuda") / inner ** 0.5
    if kind == "bf16":
        return ops.MoEWeights(w13.bfloat16(), w2.bfloat16())
    if kind == "w4":
        (q13, s13, z13), (q2, s2, z2) = (ops.quantize_weight_w4(w, 64, asymmetric=True) for w in (w13, w2))
        return ops.MoEWeights(q13, q2, s13, s2, z13, z2)
    (q13, s13), (q2, s2) = (ops.quantize_weight_block_fp8(w) for w in (w13, w2))
    return ops.MoEWeights(q13, q2, s13, s2)


class DecodeTail:
    """Weights, request state and the step; ``step`` works on fixed buffers
    only, so it can be captured."""

    def __init__(self, requests=4, hidden=1024, experts=32, top_k=4, inner=512, shared=1024, vocab=32000,
                 max_len=256, weights="w4", seed=0):
        torch.manual_seed(seed)
        self.top_k = top_k
        self.embedding = torch.randn((vocab, hidden), device="cuda").bfloat16()
        self.router = torch.randn((experts, hidden), device="cuda") / hidden ** 0.5
        self.router_bias = torch.randn(experts, device="cuda") * 0.05
        self.experts = random_experts(weights, (experts,), hidden, inner)
        self.shared = random_experts(weights, (), hidden, shared)
        self.vocab_q, self.vocab_s, _ = ops.quantize_weight_w4(torch.randn((vocab, hidden), device="cuda") / hidden ** 0.5, 128)
        # a request's tokens: its prompt (one token here), then its answer
        self.token_ids = torch.full((requests, max_len), -1, dtype=torch.int32, device="cuda")
        self.token_ids[:, 0] = torch.randint(0, vocab, (requests,), device="cuda")
        self.prompt_lens = torch.ones(requests, dtype=torch.int32, device="cuda")
        self.seq_lens = self.prompt_lens.clone()
        self.repetition = torch.full((requests,), 1.1, device="cuda")
        self.frequency = torch.full((requests,), 0.2, device="cuda")
        self.presence = torch.full((requests,), 0.1, device="cuda")
        self.bias_ids = torch.tensor([[7, -1]], dtype=torch.int32, device="cuda").repeat(requests, 1)
        self.bias_values = torch.full((requests, 2), 0.5, device="cuda")
        # bit v of a row's mask: token v is allowed; here all of them
        self.allowed = torch.full((requests, (vocab + 31) // 32), -1, dtype=torch.int32, device="cuda")
        self.logits = torch.empty((requests, vocab), device="cuda", dtype=torch.bfloat16)

    def forbid(self, request: int, tokens) -> None:
        """Clears the tokens' bits of a request's mask."""
        words = self.allowed[request].cpu()
        for v in tokens:
            bit = v % 32
            words[v // 32] &= ~(1 << bit) if bit < 31 else 0x7FFFFFFF
        self.allowed[request] = words.cuda()

    def scores(self) -> torch.Tensor:
        """The logits of each request's last token, penalised and masked."""
        last = self.token_ids.gather(1, (self.seq_lens - 1).long().unsqueeze(1)).squeeze(1)
        x = self.embedding[last.long()]
        x = x + ops.moe_decode(x, self.router, self.experts, self.top_k, score="sigmoid", router_bias=self.router_bias,
                               routed_scale=2.5, shared=self.shared)
        ops.w4_linear(x, self.vocab_q, self.vocab_s, out=self.logits)
        return ops.apply_logit_penalties(self.logits, self.token_ids, self.prompt_lens, self.seq_lens,
                                         repetition=self.repetition, frequency=self.frequency, presence=self.presence,
                                         bias_ids=self.bias_ids, bias_values=self.bias_values, allowed_bitmask=self.allowed)

    def step(self) -> None:
        """Appends a token to each history; of a full one it replaces the last."""
        token = self.scores().argmax(1)
        room = self.token_ids.shape[1]
        self.token_ids.scatter_(1, self.seq_lens.long().clamp(max=room - 1).unsqueeze(1), token.int().unsqueeze(1))
        self.seq_lens.add_(1).clamp_(max=room)

    def capture(self) -> torch.cuda.CUDAGraph:
        """A graph of one step; capturing leaves the histories as they are."""
        ids, lens = self.token_ids.clone(), self.seq_lens.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self.step()
        torch.cuda.current_stream().wait_stream(side)
        self.token_ids.copy_(ids)
        self.seq_lens.copy_(lens)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.step()
        return graph


def main(argv=None) -> list[list[int]]:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--requests", type=int, default=4)
    p.add_argument("--steps", type=int, default=32)
    p.add_argument("--weights", choices=["bf16", "fp8", "w4"], default="w4")
    p.add_argument("--vocab", type=int, default=32000)
    args = p.parse_args(argv)
    tail = DecodeTail(requests=args.requests, weights=args.weights, vocab=args.vocab, max_len=args.steps + 1)
    graph = tail.capture()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(args.steps):
        graph.replay()
    end.record()
    answers = tail.token_ids[:, 1:].tolist()
    for i, answer in enumerate(answers):
        print(f"request {i}: {answer}")
    print(f"{begin.elapsed_time(end) * 1e3 / max(args.steps, 1):.1f} us a step of {args.requests} tokens")
    return answers


if __name__ == "__main__":
    main()
