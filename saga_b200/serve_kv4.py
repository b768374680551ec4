"""One attention layer served from the paged 4-bit cache: an example of the operators of saga_b200.kv4 together.

    python -m saga_b200.serve_kv4 --requests 8 --prompt 4096 --steps 64 --top 16

Requests of ragged prompt lengths are admitted into one pool: their pages, slots
and positions come from ``page_tables``, and ``kv4_write`` quantises their keys
and values. Decode steps (tables, write, attention; with --top also the
selection of blocks) then run as one CUDA graph, replayed once per token; nothing
in it reads a length on the host. Half way one request finishes: its pages go
back to the free ring, and a new prompt is admitted in its row. At the end the
last step's output is compared with the 16-bit dense decode of the same keys and
values, and one JSON line says how far apart they are and what the step takes.
Queries, keys and values are synthetic (a layer's projections are not part of
this library).
"""
from __future__ import annotations

import argparse
import json
import random

import torch

from . import kv4, ops


class Layer:
    """The serving state of one layer: pool, page table, lengths and the free ring."""

    def __init__(self, rows: int, width: int, num_pages: int, page_len: int, heads, head_dim: int, dtype, device):
        self.hq, self.hk, self.hv = heads
        self.rows, self.d, self.dtype, self.device = rows, head_dim, dtype, device
        i32 = dict(dtype=torch.int32, device=device)
        self.pool = kv4.Kv4Pool(num_pages, page_len, self.hk, self.hv, head_dim, device=device, bounds=True)
        self.table = torch.full((rows, width), -1, **i32)
        self.lens = torch.zeros(rows, **i32)
        self.free = torch.arange(num_pages, **i32)
        self.free_state = torch.tensor([0, num_pages], **i32)

    def place(self, new_lens: torch.Tensor, num_tokens: int) -> kv4.PageStep:
        """Pages and slots for the next tokens of every row (lengths advance in place)."""
        return kv4.page_tables(self.table, self.lens, new_lens, self.free, self.free_state, num_tokens,
                               self.pool.page_len, lens_out=self.lens, free_state_out=self.free_state)

    def admit(self, row: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """A new request's prompt, [n, H, D], in an idle row."""
        new = torch.zeros(self.rows, dtype=torch.int32)
        new[row] = k.shape[0]
        step = self.place(new.to(self.device), k.shape[0])
        kv4.kv4_write(self.pool, k, v, step.slots)

    def finish(self, row: int) -> None:
        """Returns a request's pages to the free ring."""
        new = torch.zeros(self.rows, dtype=torch.int32)
        new[row] = -1
        self.place(new.to(self.device), 0)

    def step(self, q, k, v, ones, top: int = 0) -> torch.Tensor:
        """One token for every row: q [B, Hq, 1, D], k [B, Hk, D], v [B, Hv, D]."""
        place = self.place(ones, self.rows)
        kv4.kv4_write(self.pool, k, v, place.slots)
        if not top:
            return kv4.kv4_decode(q, self.pool, self.table, self.lens)
        blocks, counts = kv4.kv4_select(q, self.pool, self.table, self.lens, top)
        return kv4.kv4_decode(q, self.pool, self.table, self.lens, blocks=blocks, counts=counts)


def serve(requests: int = 8, prompt: int = 4096, steps: int = 64, top: int = 0, page_len: int = 64, heads=(12, 1, 2),
          head_dim: int = 128, seed: int = 0, device: str = "cuda") -> dict:
    """Runs the loop of the module's description and returns what it measured."""
    rng = random.Random(seed)
    g = torch.Generator(device=device).manual_seed(seed)
    dtype = torch.bfloat16
    hq, hk, hv = heads
    prompts = [rng.randint(max(1, prompt // 2), prompt) for _ in range(requests + 1)]
    width = (max(prompts) + steps) // page_len + 2
    layer = Layer(requests, width, width * requests, page_len, heads, head_dim, dtype, device)

    def rows(n, h):
        return torch.randn((n, h, head_dim), generator=g, device=device).to(dtype)

    history = []  # the 16-bit rows of every request, for the comparison at the end
    for b in range(requests):
        history.append([rows(prompts[b], hk), rows(prompts[b], hv)])
        layer.admit(b, *history[b])

    q = torch.zeros((requests, hq, 1, head_dim), dtype=dtype, device=device)
    k, v = rows(requests, hk), rows(requests, hv)
    ones = torch.ones(requests, dtype=torch.int32, device=device)
    state = (layer.table, layer.lens, layer.free, layer.free_state, layer.pool.k, layer.pool.v, layer.pool.k_lo,
             layer.pool.k_hi)
    saved = [t.clone() for t in state]
    stream, graph = torch.cuda.Stream(device=device), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer.step(q, k, v, ones, top)  # allocates the workspace
        for t, s in zip(state, saved):
            t.copy_(s)
        with torch.cuda.graph(graph, stream=stream):
            out = layer.step(q, k, v, ones, top)
    torch.cuda.current_stream().wait_stream(stream)
    del saved

    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    total_ms = 0.0
    for i in range(steps):
        if i == steps // 2:
            layer.finish(0)
            history[0] = [rows(prompts[-1], hk), rows(prompts[-1], hv)]
            layer.admit(0, *history[0])
        q.copy_(torch.randn(q.shape, generator=g, device=device))
        k.copy_(rows(requests, hk))
        v.copy_(rows(requests, hv))
        begin.record()
        graph.replay()
        end.record()
        end.synchronize()
        total_ms += begin.elapsed_time(end)
        for b in range(requests):
            history[b] = [torch.cat((history[b][0], k[b:b + 1])), torch.cat((history[b][1], v[b:b + 1]))]

    # the same attention over the 16-bit rows, request by request
    worst, cosine = 0.0, 1.0
    for b in range(requests):
        kb, vb = (t.transpose(0, 1)[None].contiguous() for t in history[b])
        ref = ops.dense_decode(q[b:b + 1], kb, vb).float()
        got = out[b:b + 1].float()
        worst = max(worst, float((got - ref).norm() / ref.norm()))
        cosine = min(cosine, float(torch.nn.functional.cosine_similarity(got.flatten(), ref.flatten(), dim=0)))
    lens = layer.lens.tolist()
    held = sum((n + page_len - 1) // page_len for n in lens)
    packed = held * (layer.pool.k[0].numel() + layer.pool.v[0].numel())
    wide = sum(lens) * (hk + hv) * head_dim * 2
    return dict(lens=lens, expected_lens=[t[0].shape[0] for t in history], pages_held=held,
                pages_free=int(layer.free_state[1]), pages=layer.pool.num_pages, cache_bytes=packed,
                cache_bytes_16bit=wide, us_per_step=round(total_ms / steps * 1e3, 2),
                tokens_per_s=round(requests * steps / total_ms * 1e3), top=top,
                relative_error_to_16bit=round(worst, 4), cosine_to_16bit=round(cosine, 4),
                status=ops.read_status(device))


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=4096, help="longest prompt")
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--top", type=int, default=0, help="blocks per request and key head (0: all)")
    ap.add_argument("--page-len", type=int, default=64)
    ap.add_argument("--heads", type=int, nargs=3, default=(12, 1, 2), metavar=("HQ", "HK", "HV"))
    ap.add_argument("--head-dim", type=int, default=128)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    print(json.dumps(serve(a.requests, a.prompt, a.steps, a.top, a.page_len, tuple(a.heads), a.head_dim, a.seed)))


if __name__ == "__main__":
    main()
