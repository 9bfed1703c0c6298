"""A ragged batch through the attention operators, as a serving and as a training program use them.

Serving: requests with prompts of different lengths are admitted together.  Every step is planned on the GPU from the
requests' lengths (pages from a free list, a slot for each new token), its keys and values go to their slots, and its
rows attend: prompts packed to themselves, then single tokens to the pages, then a tree of drafted tokens whose longest
right branch is kept.  At the end each request's outputs are compared with plain attention over its whole sequence.

Training: the same layer with its gradients, as an autograd function, on packed examples.

    python examples/ragged_batch.py
"""
from __future__ import annotations

import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "luisacompute-parallelprimitive_amd"))
import lcpp_hip as hip  # noqa: E402

HEADS, KV_HEADS, DIM, WIDTH, PAGE = 8, 2, 64, 256, 16


class Layer:
    """Projections of one attention layer; a token's input is its row of `embedding`."""

    def __init__(self, vocabulary: int = 1000, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        make = lambda *shape: torch.randn(*shape, device="cuda", generator=g)
        self.embedding = make(vocabulary, WIDTH).bfloat16()
        self.fused = (make(WIDTH, (HEADS + 2 * KV_HEADS) * DIM) * WIDTH ** -0.5).bfloat16()

    def rows(self, tokens):
        """Queries, keys and values of tokens: views into one product."""
        x = (self.embedding[tokens] @ self.fused).view(-1, HEADS + 2 * KV_HEADS, DIM)
        return x[:, :HEADS], x[:, HEADS:HEADS + KV_HEADS], x[:, HEADS + KV_HEADS:]


class Cache:
    """Pages of keys and values for a fixed number of requests, and the buffers of a step."""

    def __init__(self, requests: int, longest: int, step_tokens: int):
        ints = lambda *shape, dtype=torch.int32: torch.zeros(*shape, dtype=dtype, device="cuda")
        width = -(-longest // PAGE)
        self.requests, self.longest = requests, longest
        self.keys = torch.zeros(requests * width, PAGE, KV_HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        self.values = torch.zeros_like(self.keys)
        self.free = list(range(requests * width))
        self.table, self.lengths = ints(requests, width), ints(requests)
        self.offsets, self.kv_lengths, self.counts = ints(requests + 1), ints(requests), ints(2)
        self.request, self.position = ints(step_tokens), ints(step_tokens)
        self.slot = ints(step_tokens, dtype=torch.int64)

    def append(self, new_lengths, key, value):
        """Plans a step of `new_lengths` tokens a request and writes their keys and values."""
        tokens = key.shape[0]
        free = torch.tensor(self.free, dtype=torch.int32, device="cuda")
        hip.page_plan(self.lengths, new_lengths, PAGE, free, self.table, self.offsets, self.kv_lengths,
                      self.request[:tokens], self.position[:tokens], self.slot[:tokens], self.counts)
        planned, taken = self.counts.tolist()
        assert planned == tokens and taken <= len(self.free), "no pages left"
        del self.free[:taken]
        hip.paged_write("bf16", key, value, self.slot[:tokens], self.keys, self.values)

    def keep(self, lengths):
        """The requests' lengths from now on; pages past them go back to the free list."""
        held = (self.kv_lengths + PAGE - 1) // PAGE - (lengths + PAGE - 1) // PAGE
        for r, count in enumerate(held.tolist()):
            last = int((self.kv_lengths[r] + PAGE - 1) // PAGE)
            self.free[:0] = self.table[r, last - count:last].tolist()
        self.lengths.copy_(lengths)

    def attend(self, q, tree=None):
        out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
        hip.attention_paged("bf16", q, self.keys, self.values, self.table, self.offsets, self.kv_lengths, out, tree=tree,
                            max_kv_length=self.longest)
        return out


def plain(layer, tokens):
    """Causal attention over one whole sequence in 32 bits."""
    q, k, v = (x.float().transpose(0, 1) for x in layer.rows(torch.tensor(tokens, device="cuda")))
    k, v = k.repeat_interleave(HEADS // KV_HEADS, 0), v.repeat_interleave(HEADS // KV_HEADS, 0)
    scores = (q @ k.transpose(1, 2)) * DIM ** -0.5
    hidden = torch.ones(len(tokens), len(tokens), dtype=torch.bool, device="cuda").triu(1)
    return (scores.masked_fill(hidden, -torch.inf).softmax(-1) @ v).transpose(0, 1)


def serve(prompt_lengths=(37, 1, 150, 16, 64), decoded: int = 5) -> float:
    """Prompts, single tokens, and a tree; the largest difference from plain attention."""
    g = torch.Generator().manual_seed(1)
    draw = lambda n: torch.randint(0, 1000, (n,), generator=g).tolist()
    layer, count = Layer(), len(prompt_lengths)
    texts, outputs = [draw(n) for n in prompt_lengths], [[] for _ in prompt_lengths]
    cache = Cache(count, max(prompt_lengths) + decoded + 16, max(sum(prompt_lengths), 5 * count))
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")

    # Prompts: packed attention among themselves, their keys and values into pages for later.
    q, k, v = layer.rows(torch.tensor(sum(texts, []), device="cuda"))
    cache.append(ints([len(t) for t in texts]), k, v)
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    hip.attention_packed("bf16", q, k, v, cache.offsets, cache.offsets, out)
    for r, rows in enumerate(out.split([len(t) for t in texts])):
        outputs[r].append(rows)
    cache.keep(cache.kv_lengths.clone())

    # One token a request and step.
    for _ in range(decoded):
        step = draw(count)
        q, k, v = layer.rows(torch.tensor(step, device="cuda"))
        cache.append(ints([1] * count), k, v)
        out = cache.attend(q)
        for r in range(count):
            texts[r].append(step[r])
            outputs[r].append(out[r:r + 1])
        cache.keep(cache.kv_lengths.clone())

    # A tree of five drafted tokens: 0 - 1 - 3, 0 - 2, 1 - 4.  Request r keeps the branch 0 - 1 - 3 or 0 alone.
    parents = [-1, 0, 0, 1, 1]
    words = []
    for i, parent in enumerate(parents):
        words.append((words[parent] if parent >= 0 else 0) | 1 << i)
    drafts = [draw(5) for _ in range(count)]
    q, k, v = layer.rows(torch.tensor(sum(drafts, []), device="cuda"))
    cache.append(ints([5] * count), k, v)
    out = cache.attend(q, torch.tensor(words * count, dtype=torch.int64, device="cuda"))
    branches = [[0, 1, 3] if r % 2 == 0 else [0] for r in range(count)]
    kept = []
    for r, branch in enumerate(branches):
        texts[r] += [drafts[r][i] for i in branch]
        outputs[r].append(out[5 * r:5 * r + 5][branch])
        kept.append(len(texts[r]))
    cache.keep(ints(kept))
    # The branch's keys and values move up behind the context: rows 0, 1, 3 of each request to its first places.
    rows = torch.tensor([5 * r + i for r, branch in enumerate(branches) for i in branch], device="cuda")
    to = torch.cat([cache.slot[5 * r:5 * r + len(branch)] for r, branch in enumerate(branches)])
    hip.paged_write("bf16", k[rows], v[rows], to, cache.keys, cache.values)

    # One more token each, over the moved branch.
    step = draw(count)
    q, k, v = layer.rows(torch.tensor(step, device="cuda"))
    cache.append(ints([1] * count), k, v)
    out = cache.attend(q)
    worst = 0.0
    for r in range(count):
        texts[r].append(step[r])
        got = torch.cat(outputs[r] + [out[r:r + 1]]).float()
        worst = max(worst, float((got - plain(layer, texts[r])).abs().max()))
    return worst


class PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets):
        out, lse = torch.empty_like(q), torch.empty(q.shape[1], q.shape[0], device=q.device)
        hip.attention_packed("bf16", q, k, v, offsets, offsets, out, lse)
        ctx.save_for_backward(q, k, v, out, lse, offsets)
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse, offsets = ctx.saved_tensors
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
        hip.attention_packed_backward("bf16", q, k, v, out, lse, dout.contiguous(), offsets, offsets, dq, dk, dv)
        return dq, dk, dv, None


def train(lengths=(90, 33, 200), steps: int = 12) -> list:
    """Fits the layer's projections to fixed targets on packed examples; the loss of every step."""
    g = torch.Generator(device="cuda").manual_seed(2)
    layer = Layer(seed=3)
    tokens = torch.randint(0, 1000, (sum(lengths),), device="cuda", generator=g)
    target = torch.randn(sum(lengths), HEADS, DIM, device="cuda", generator=g) * 0.3
    offsets = torch.tensor([0, *lengths], device="cuda").cumsum(0).int()
    weight = layer.fused.float().requires_grad_()
    optimizer, losses = torch.optim.Adam([weight], lr=2e-3), []
    for _ in range(steps):
        layer.fused = weight.bfloat16()
        loss = (PackedAttention.apply(*layer.rows(tokens), offsets).float() - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses


if __name__ == "__main__":
    print(f"serving: largest difference from plain attention {serve():.4f}")
    losses = train()
    print(f"training: loss {losses[0]:.4f} -> {losses[-1]:.4f}")
