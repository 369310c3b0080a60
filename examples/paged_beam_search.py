"""Beam search of a batch of requests over a paged 8-bit cache: the serving operators together, as a runtime calls them.

    python examples/paged_beam_search.py [--requests 3] [--width 4] [--steps 12]

A small decoder with random weights in the library's block formats: Q/K/V, output, feed-forward and head products in Q8_0 and
Q4_K on the repacked GEMM, SwiGLU fused into its quantizer. Each request is a group of `width` rows. A step is

    jk_paged_extend      pages, slots and positions of the step's tokens
    per layer            products, rotary embedding, jk_kv_append_q8, jk_attn_q8, feed-forward
    jk_beam_select       the group's next hypotheses
    jk_paged_reorder     their rows of the tables, and jk_kv_reorder_q8 in each layer's cache

The prompt goes through the first row of each group alone; the first reordering hands it to the others (full pages are
shared, the open one is copied). Norms and the rotary embedding are the runtime's own, in torch.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jero-kernels-rvv_amd"))

import jk  # noqa: E402
from jk import synth  # noqa: E402

DEV = "cuda"


def ints(*shape, value=0):
    return torch.full(shape, value, dtype=torch.int32, device=DEV)


class Product:
    """A quantized matrix and its products with a batch of tokens."""

    def __init__(self, quant, rows, cols, seed):
        view = jk.TensorView(f"w{seed}", quant, (rows, cols), synth.gguf_weights(quant, rows, cols, seed=seed))
        self.w, self.rows, self.cols = jk.Weight(view, rows, cols), rows, cols

    def __call__(self, act):
        y = torch.empty((act.m, self.rows), device=DEV)
        jk.dev_gemm_repacked(self.w, act, y, y.numel(), 0, self.rows, stream=torch.cuda.current_stream().cuda_stream)
        return y


def quantized(x, up=None):
    """The product's activation of a batch of tokens; with `up`, of SwiGLU(x, up)."""
    m, k = x.shape
    store = torch.empty(jk.act_q8_bytes(m, k), dtype=torch.uint8, device=DEV)
    act = jk.act_q8_bind(store, store.numel(), m, k)
    act.storage = store
    s = torch.cuda.current_stream().cuda_stream
    if up is None:
        jk.dev_quantize_act_q8(x.contiguous(), m, k, act, stream=s)
    else:
        jk.dev_quantize_act_q8_gated(jk.ACT_SWIGLU, x, up, m, k, act, stream=s)
    return act


def normed(x):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5)


def rotated(x, positions):
    """Rotary embedding of [tokens][heads][dim] by each token's position."""
    half = x.shape[-1] // 2
    angle = positions.float()[:, None] * torch.pow(10000.0, -torch.arange(half, device=DEV) / half)[None]
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


class Decoder:
    def __init__(self, layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=1000, pages=256, page=16):
        self.heads, self.kv, self.hd, self.vocab = heads, kv_heads, head_dim, vocab
        g = torch.Generator(device=DEV).manual_seed(1)
        self.embed = torch.randn((vocab, hidden), generator=g, device=DEV)
        self.layers = []
        for i in range(layers):
            p = [Product(jk.Q8_0, (heads + 2 * kv_heads) * head_dim, hidden, 10 * i + 1),
                 Product(jk.Q8_0, hidden, heads * head_dim, 10 * i + 2), Product(jk.Q4_K, ffn, hidden, 10 * i + 3),
                 Product(jk.Q4_K, ffn, hidden, 10 * i + 4), Product(jk.Q8_0, hidden, ffn, 10 * i + 5)]
            codes = [torch.zeros((pages, kv_heads, page, head_dim), dtype=torch.int8, device=DEV) for _ in range(2)]
            self.layers.append((p, jk.kv_q8(*codes, *(torch.zeros((pages, kv_heads), device=DEV) for _ in range(2)))))
        self.head = Product(jk.Q8_0, vocab, hidden, 99)

    def __call__(self, tokens, batch, last):
        """Logits of the tokens at `last` of a planned step; their keys and values go into the caches."""
        stream = torch.cuda.current_stream().cuda_stream
        n = tokens.numel()
        slots, positions = batch.slots[:n], batch.positions[:n]
        x = self.embed[tokens.long()]
        for (qkv, out, gate, up, down), cache in self.layers:
            y = qkv(quantized(normed(x))).view(n, -1, self.hd)
            q = rotated(y[:, :self.heads], positions)
            k = rotated(y[:, self.heads:self.heads + self.kv], positions)
            v = y[:, self.heads + self.kv:].contiguous()
            jk.dev_kv_append_q8(cache, k, v, slots, stream=stream)
            o = torch.empty_like(q)
            a = jk.attn_q8_args(q, o, batch.q_start, batch.lens, batch.table, max_new=batch.max_new,
                                max_len=batch.max_len, scale=self.hd ** -0.5)
            ws = torch.empty(max(16, jk.attn_q8_workspace_bytes(cache, a)), dtype=torch.uint8, device=DEV)
            jk.dev_attn_q8(cache, a, ws, stream=stream)
            x = x + out(quantized(o.view(n, -1)))
            act = quantized(normed(x))
            x = x + down(quantized(gate(act), up(act)))
        return self.head(quantized(normed(x[last])))


class Batch:
    """The pages of groups of `width` rows, and the plan of the step in hand."""

    def __init__(self, rows, columns, pages, page, tokens):
        self.lens, self.table, self.owned = ints(rows), ints(rows, columns), ints(rows, columns)
        self.free, self.n_free, self.status = ints(pages), ints(1), ints(1)
        self.q_start, self.slots, self.positions, self.of = ints(rows + 1), ints(tokens), ints(tokens), ints(tokens)
        self.paged = jk.paged(self.lens, self.table, self.owned, self.free, self.n_free, page)
        self.step = jk.paged_step(self.q_start, self.slots, self.positions, self.of, self.status)
        jk.dev_paged_reset(self.paged, stream=torch.cuda.current_stream().cuda_stream)

    def extend(self, n_new, max_new, max_len):
        self.max_new, self.max_len = max_new, max_len
        jk.dev_paged_extend(self.paged, n_new, self.step, stream=torch.cuda.current_stream().cuda_stream)

    def reorder(self, parents, width, caches):
        s = torch.cuda.current_stream().cuda_stream
        jk.dev_paged_reorder(self.paged, parents, width, self.status, stream=s)
        for cache in caches:
            jk.dev_kv_reorder_q8(cache, self.paged, parents, width, self.status, stream=s)


def search(model, prompts, width, steps, eos=2, page=16, seen=None):
    """The `width` best continuations of each prompt, (scores, tokens [groups][width][steps]). seen(event, **what):
    called after each selection and each reordering."""
    groups, longest = len(prompts), max(len(p) for p in prompts)
    rows, total = groups * width, sum(len(p) for p in prompts)
    stream = torch.cuda.current_stream().cuda_stream
    pages = model.layers[0][1].n_pages
    batch = Batch(rows, -(-(longest + steps) // page) + 1, pages, page, max(total, rows))
    caches = [c for _, c in model.layers]

    # prompts through the first row of each group
    n_new = ints(rows)
    n_new[::width] = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=DEV)
    batch.extend(n_new, longest, longest)
    tokens = torch.tensor(sum(prompts, []), dtype=torch.int32, device=DEV)
    logits = model(tokens, batch, (torch.cumsum(n_new, 0) - 1)[::width].long()).repeat_interleave(width, 0)

    # one hypothesis a group at first: the others' scores are -inf
    scores = torch.full((groups, width), -torch.inf, device=DEV)
    scores[:, 0] = 0
    done, best = ints(groups, width), torch.empty_like(scores)
    parents, chosen, ended = ints(groups, width), ints(groups, width), ints(groups, width)
    history, one = ints(groups, width, 0), ints(rows, value=1)
    for i in range(steps):
        args = jk.beam_args(logits, scores, done, best, parents, chosen, ended, eos=eos)
        ws = torch.empty(jk.beam_workspace_bytes(args), dtype=torch.uint8, device=DEV)
        jk.dev_beam_select(args, ws, stream=stream)
        if seen:
            seen("selected", logits=logits, scores=scores, done=done, best=best, parents=parents, chosen=chosen, eos=eos)
        history = torch.cat([history.gather(1, parents.long()[..., None].expand_as(history)), chosen[..., None]], 2)
        scores, done = best.clone(), ended.clone()
        if i + 1 == steps:
            break
        if seen:
            seen("reordering", batch=batch, caches=caches, parents=parents, width=width)
        batch.reorder(parents, width, caches)
        if seen:
            seen("reordered", batch=batch, caches=caches, parents=parents, width=width)
        batch.extend(one, 1, longest + i + 1)
        logits = model(chosen.view(-1), batch, slice(None))
    if int(batch.status):
        raise RuntimeError(f"the step did not fit: status {int(batch.status)}")
    jk.dev_paged_release(batch.paged, one, stream=stream)
    if int(batch.n_free) != pages:
        raise RuntimeError("pages were lost")
    return scores, history


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=3)
    ap.add_argument("--width", type=int, default=4)
    ap.add_argument("--steps", type=int, default=12)
    a = ap.parse_args()
    jk.init(0)
    model = Decoder(pages=max(256, a.requests * a.width * (4 + a.steps // 16)))
    gen = torch.Generator().manual_seed(7)
    prompts = [torch.randint(3, model.vocab, (5 + 17 * r % 40,), generator=gen).tolist() for r in range(a.requests)]
    scores, history = search(model, prompts, a.width, a.steps)
    for r in range(a.requests):
        print(f"request {r} ({len(prompts[r])} tokens of prompt)")
        for b in range(a.width):
            print(f"  {scores[r, b].item():9.4f}  {history[r, b].tolist()}")


if __name__ == "__main__":
    main()
