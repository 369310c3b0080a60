"""Performance cases of the operators that serve a batch from a paged attention cache held in 8 bits.

A runtime that decodes a batch of requests calls them between the products of each layer:

  tables  jk_paged_extend: which page and slot each new token of a step goes to
  append  jk_kv_append_q8: the layer's new keys and values into the cache, one scale per page and head
          (read back with jk_kv_read_q8, as a runtime does that moves a request's pages away)
  attn    jk_attn_q8: the layer's attention over the cache, one token a request up to a whole prompt
  beam    jk_beam_select and jk_paged_reorder: the next hypotheses of beam search, and their cache rows

Head counts and vocabulary are Llama-3-8B's (32 query and 8 key heads of 128, 128256 tokens) or generic; pages hold
16 to 128 tokens. draw() spreads the sizes over the ranges in between. Queries and keys are normal with a few
channels several times larger, as attention's are; pages lie in no order, as after a while of serving.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY = 2.0 ** -119  # largest values below this are stored as zeros


def _jk():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jero-kernels-rvv_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import jk

    return jk


def listed():
    return [
        # one step of four chats: the smallest plan
        {"name": "tables_step_b4", "kind": "tables", "requests": 4, "prompt": 0, "held": 3000, "page": 64},
        # a step that takes in the prompts of 96 requests of very different lengths
        {"name": "tables_prompts_b96", "kind": "tables", "requests": 96, "prompt": 1024, "held": 2000, "page": 32},
        # the new token of 48 concurrent requests, in the middle of their pages
        {"name": "append_step_b48", "kind": "append", "dtype": "bf16", "requests": 48, "prompt": 0, "held": 8000,
         "page": 64, "kv_heads": 8, "head_dim": 128},
        # the prompts of 9 requests into the cache, activations in f32 as the library's products leave them
        {"name": "append_prompts_f32", "kind": "append", "dtype": "f32", "requests": 9, "prompt": 2048, "held": 1000,
         "page": 64, "kv_heads": 8, "head_dim": 128},
        # a small model's decode step for three short chats in f32: latency alone
        {"name": "attn_step_small_f32", "kind": "attn", "dtype": "f32", "requests": 3, "new": 1, "held": 700,
         "page": 16, "heads": 14, "kv_heads": 2, "head_dim": 64, "window": 0, "ragged": True},
        # one request with a long document: few rows over a long axis
        {"name": "attn_step_32k", "kind": "attn", "dtype": "f32", "requests": 1, "new": 1, "held": 32768,
         "page": 64, "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0, "ragged": False},
        # the decode step of 64 concurrent requests of very different lengths
        {"name": "attn_step_b64", "kind": "attn", "dtype": "bf16", "requests": 64, "new": 1, "held": 8192,
         "page": 64, "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0, "ragged": True},
        # a step that checks five drafted tokens of each of 16 requests, with a sliding window
        {"name": "attn_draft_window", "kind": "attn", "dtype": "f16", "requests": 16, "new": 5, "held": 9001,
         "page": 128, "heads": 24, "kv_heads": 8, "head_dim": 96, "window": 4096, "ragged": True},
        # chunks of three prompts in f32, on top of what the cache holds of them
        {"name": "attn_chunks_f32", "kind": "attn", "dtype": "f32", "requests": 3, "new": 511, "held": 4000,
         "page": 32, "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0, "ragged": True},
        # one whole prompt: the largest call
        {"name": "attn_prompt_4096", "kind": "attn", "dtype": "bf16", "requests": 1, "new": 4096, "held": 0,
         "page": 64, "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0, "ragged": False},
        # one request's beam search over a small vocabulary
        {"name": "beam_w4", "kind": "beam", "dtype": "f32", "groups": 1, "width": 4, "vocab": 32000, "held": 500,
         "page": 64},
        # 16 requests with eight hypotheses each at Llama-3's vocabulary
        {"name": "beam_g16_w8", "kind": "beam", "dtype": "f32", "groups": 16, "width": 8, "vocab": 128256,
         "held": 2000, "page": 64},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ranges that needs no more than the largest listed ones."""
    most = [max(w[i] for w in map(work, listed())) for i in ("bytes", "flops")]
    while True:
        case = _drawn(rng)
        if work(case)["bytes"] <= most[0] and work(case)["flops"] <= most[1]:
            return case


def _drawn(rng):
    kind = rng.choice(["tables", "append", "step", "step", "draft", "prompt", "prompt", "beam", "beam"])
    page = rng.choice([16, 32, 64, 128])
    if kind in ("tables", "append"):
        prompts = rng.random() < 0.5
        c = {"kind": kind, "requests": _log_int(rng, 1, 16 if prompts else 400),
             "prompt": _log_int(rng, 16, 2048) if prompts else 0, "held": _log_int(rng, 1, 8000), "page": page}
        if kind == "append":
            c.update(dtype=rng.choice(list(TYPES)), kv_heads=rng.choice([1, 2, 4, 8]),
                     head_dim=rng.choice([64, 80, 96, 128, 256]))
        return c
    if kind == "beam":
        return {"kind": "beam", "dtype": rng.choice(list(TYPES)), "groups": _log_int(rng, 1, 16),
                "width": rng.choice([2, 3, 4, 5, 8]), "vocab": _log_int(rng, 1000, 128256),
                "held": _log_int(rng, 10, 4000), "page": page}
    kv = rng.choice([1, 2, 4, 8])
    c = {"kind": "attn", "dtype": rng.choice(list(TYPES)), "page": page, "kv_heads": kv,
         "heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "head_dim": rng.choice([64, 64, 80, 96, 128, 128, 128, 256]),
         "ragged": rng.random() < 0.7, "window": rng.choice([0, 0, 0, _log_int(rng, 64, 4096)])}
    if kind == "step":
        n = _log_int(rng, 1, 64)
        c.update(requests=n, new=1, held=_log_int(rng, 100, min(32768, 300000 // n)))
    elif kind == "draft":
        n = _log_int(rng, 1, 24)
        c.update(requests=n, new=rng.randint(2, 16), held=_log_int(rng, 100, min(16384, 150000 // n)))
    else:
        new = _log_int(rng, 17, 2048)
        n = _log_int(rng, 1, max(1, 2048 // new))
        c.update(requests=n, new=new, held=_log_int(rng, 1, min(8192, 4000000 // (n * new))))
    return c


# ------------------------------------------------------------------ inputs
def _generator(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 64 + salt)


def _ints(gen, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=gen, device=DEV, dtype=torch.int32)


def _lengths(case, seed, held, new):
    """Held and new tokens of the requests: the same pairs at every seed (so that sizes stay), in the seed's order."""
    fixed = _generator(0, 6)
    n = case["requests"]
    pairs = [torch.full((n,), x[0], dtype=torch.int32, device=DEV) if x[0] == x[1] else _ints(fixed, x[0], x[1], n)
             for x in (held, new)]
    order = torch.randperm(n, generator=_generator(seed, 1), device=DEV)
    return pairs[0][order], pairs[1][order]


def _pages_of(lens, page):
    return torch.div(lens + page - 1, page, rounding_mode="floor")


def _tables(lens, page, max_pages, n_pages, gen):
    """A table whose first pages are in use, in no order, and the stack of the free ones."""
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    used = _pages_of(lens, page).long()
    j = torch.arange(max_pages, device=DEV)
    live = j[None] < used[:, None]
    table = torch.full((lens.numel(), max_pages), -1, dtype=torch.int32, device=DEV)
    n_used = int(used.sum())
    table[live] = order[:n_used]
    free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    free[:n_pages - n_used] = order[n_used:]
    return table, free, torch.tensor([n_pages - n_used], dtype=torch.int32, device=DEV)


def _batch(case, seed):
    """Lengths held and new tokens of a step's requests: single tokens, or prompts of ragged lengths."""
    gen = _generator(seed, 2)
    b, page = case["requests"], case["page"]
    lens, new = _lengths(case, seed, (1, case["held"]), (1, max(1, case["prompt"])))
    if not case["prompt"] and b > 3:
        new = torch.where(lens % 7 == 1, 0, new)  # requests that wait in this step
    total = int(new.sum())
    max_pages = -(-(case["held"] + max(1, case["prompt"])) // page) + 1
    n_pages = int(_pages_of(lens + new, page).sum()) + 64
    table, free, n_free = _tables(lens, page, max_pages, n_pages, gen)
    return lens, new, total, table, free, n_free


def _channels(x, gen):
    """A few channels several times larger, the same ones for every token."""
    d = x.shape[-1]
    big = torch.randperm(d, generator=gen, device=DEV)[:max(1, d // 32)]
    x[..., big] *= 5.0
    return x


def _quantized(shape, gen, outliers):
    """Codes and scales of normal values, one scale per page and head."""
    codes = torch.empty(shape, dtype=torch.int8, device=DEV)
    scale = torch.empty(shape[:2], dtype=torch.float32, device=DEV)
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for i in range(0, shape[0], step):
        x = torch.randn((min(step, shape[0] - i),) + tuple(shape[1:]), generator=gen, device=DEV)
        if outliers is not None:
            x[..., outliers] *= 5.0
        d = x.abs().amax((2, 3)) / 127
        codes[i:i + step] = torch.round(x / d[..., None, None]).to(torch.int8)
        scale[i:i + step] = d
    return codes, scale


def prepare(case, seed):
    s = {"case": case}
    if case["kind"] == "tables":
        lens, new, total, table, free, n_free = _batch(case, seed)
        cap = total + 5  # a step is sized for some more tokens than it gets
        ints = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)  # noqa: E731
        s.update(lens=lens, new=new, table=table, free=free, n_free=n_free, cap=cap, lens_out=ints(lens.numel()),
                 n_free_out=ints(1), q_start=ints(lens.numel() + 1), slots=ints(cap), positions=ints(cap),
                 of=ints(cap), status=ints(1))
    elif case["kind"] == "append":
        lens, new, total, table, free, n_free = _batch(case, seed)
        page, kv, hd = case["page"], case["kv_heads"], case["head_dim"]
        end = lens + new
        table, _, _ = _tables(end, page, table.shape[1], free.numel(), _generator(seed, 7))
        r = torch.repeat_interleave(torch.arange(lens.numel(), device=DEV), new.long())
        pos = torch.arange(total, device=DEV) - (torch.cumsum(new, 0) - new)[r] + lens[r]
        slots = table[r, pos // page] * page + pos % page
        # what is read back: every token of the pages that the step writes to
        first = torch.where(new > 0, lens // page * page, end)
        n = (end - first).long()
        rr = torch.repeat_interleave(torch.arange(lens.numel(), device=DEV), n)
        pp = torch.arange(int(n.sum()), device=DEV) - (torch.cumsum(n, 0) - n)[rr] + first[rr]
        gen = _generator(seed, 3)
        outl = torch.randperm(hd, generator=gen, device=DEV)[:max(1, hd // 32)]
        codes_k, scale_k = _quantized((free.numel(), kv, page, hd), gen, outl)
        codes_v, scale_v = _quantized((free.numel(), kv, page, hd), gen, None)
        k = torch.randn((total, kv, hd), generator=gen, device=DEV)
        k[..., outl] *= 5.0
        v = torch.randn((total, kv, hd), generator=gen, device=DEV)
        dt = TYPES[case["dtype"]]
        read = (table[rr, pp // page] * page + pp % page).to(torch.int32)
        s.update(k=k.to(dt), v=v.to(dt), slots=slots.to(torch.int32), read=read, codes_k=codes_k, codes_v=codes_v,
                 scale_k=scale_k, scale_v=scale_v,
                 k_out=torch.empty((read.numel(), kv, hd), dtype=torch.float32, device=DEV),
                 v_out=torch.empty((read.numel(), kv, hd), dtype=torch.float32, device=DEV))
    elif case["kind"] == "attn":
        gen = _generator(seed, 4)
        b, page, kv, hd = case["requests"], case["page"], case["kv_heads"], case["head_dim"]
        held, new = _lengths(case, seed, (case["held"] // 8 if case["ragged"] else case["held"], case["held"]),
                             (case["new"] // 3 if case["ragged"] and case["new"] > 16 else case["new"], case["new"]))
        lens = held + new
        q_start = torch.zeros(b + 1, dtype=torch.int32, device=DEV)
        q_start[1:] = torch.cumsum(new, 0)
        total, max_len, max_new = int(q_start[-1]), int(lens.max()), int(new.max())
        n_pages = int(_pages_of(lens, page).sum()) + 3
        table, _, _ = _tables(lens, page, -(-max_len // page) + 1, n_pages, gen)
        outl = torch.randperm(hd, generator=gen, device=DEV)[:max(1, hd // 32)]
        codes_k, scale_k = _quantized((n_pages, kv, page, hd), gen, outl)
        codes_v, scale_v = _quantized((n_pages, kv, page, hd), gen, None)
        q = torch.randn((total, case["heads"], hd), generator=gen, device=DEV).to(TYPES[case["dtype"]])
        s.update(q=q, q_start=q_start, lens=lens, table=table, codes_k=codes_k, codes_v=codes_v, scale_k=scale_k,
                 scale_v=scale_v, out=torch.empty_like(q), max_len=max_len, max_new=max_new)
    else:
        gen = _generator(seed, 5)
        g, w, v, page = case["groups"], case["width"], case["vocab"], case["page"]
        logits = torch.randn((g * w, v), generator=gen, device=DEV) * 2.5
        likely = torch.randint(0, v, (g * w, 12), generator=gen, device=DEV)
        logits.scatter_add_(1, likely, torch.rand((g * w, 12), generator=gen, device=DEV) * 9)
        scores = torch.sort(torch.rand((g, w), generator=gen, device=DEV) * -6 - 1, dim=1, descending=True)[0]
        done = (torch.rand((g, w), generator=gen, device=DEV) < 0.1).to(torch.int32)
        # the hypotheses of a group are equally long
        held, _ = _lengths({"requests": g}, seed, (max(1, case["held"] // 3), case["held"]), (0, 0))
        lens = held.repeat_interleave(w).contiguous()
        n_pages = int(_pages_of(lens, page).sum()) + 2 * g * w
        table, free, n_free = _tables(lens, page, -(-case["held"] // page) + 1, n_pages, gen)
        owned = table.clone()
        s.update(logits=logits.to(TYPES[case["dtype"]]), scores=scores, done=done, lens=lens, table=table,
                 owned=owned, free=free, n_free=n_free, eos=2, scores_out=torch.empty_like(scores),
                 parents=torch.empty_like(done), tokens=torch.empty_like(done), done_out=torch.empty_like(done),
                 lens_out=torch.empty_like(lens), table_out=torch.empty_like(table),
                 status=torch.zeros(1, dtype=torch.int32, device=DEV))
    if own:
        _handles(s)
    return s


def _handles(s):
    """The structs and workspaces that a runtime makes once for its buffers."""
    jk = _jk()
    kind, case = s["case"]["kind"], s["case"]
    if kind == "tables":
        s["paged"] = jk.paged(s["lens"], s["table"], s["table"], s["free"], s["n_free"], case["page"])
        s["step"] = jk.paged_step(s["q_start"], s["slots"], s["positions"], s["of"], s["status"])
    elif kind in ("append", "attn"):
        s["cache"] = jk.kv_q8(s["codes_k"], s["codes_v"], s["scale_k"], s["scale_v"])
    if kind == "attn":
        s["args"] = jk.attn_q8_args(s["q"], s["out"], s["q_start"], s["lens"], s["table"], max_new=s["max_new"],
                                    max_len=s["max_len"], scale=case["head_dim"] ** -0.5, window=case["window"])
        n = jk.attn_q8_workspace_bytes(s["cache"], s["args"])
        s["ws"] = torch.empty(max(16, n), dtype=torch.uint8, device=DEV)
    if kind == "beam":
        s["args"] = jk.beam_args(s["logits"], s["scores"], s["done"], s["scores_out"], s["parents"], s["tokens"],
                                 s["done_out"], eos=s["eos"])
        s["ws"] = torch.empty(jk.beam_workspace_bytes(s["args"]), dtype=torch.uint8, device=DEV)
        s["paged"] = jk.paged(s["lens"], s["table"], s["owned"], s["free"], s["n_free"], case["page"])


# ------------------------------------------------------------------ one pass
def run(s):
    return (_own if own else _plain)[s["case"]["kind"]](s)


def _own_tables(s):
    st = torch.cuda.current_stream().cuda_stream
    _jk().dev_paged_extend(s["paged"], s["new"], s["step"], s["lens_out"], s["n_free_out"], stream=st)
    return (s["q_start"], s["slots"], s["positions"], s["of"], s["table"], s["lens_out"], s["n_free_out"],
            s["status"])


def _own_append(s):
    jk, st = _jk(), torch.cuda.current_stream().cuda_stream
    jk.dev_kv_append_q8(s["cache"], s["k"], s["v"], s["slots"], stream=st)
    jk.dev_kv_read_q8(s["cache"], s["read"], s["k_out"], s["v_out"], stream=st)
    return s["scale_k"], s["scale_v"], s["k_out"], s["v_out"]


def _own_attn(s):
    _jk().dev_attn_q8(s["cache"], s["args"], s["ws"], stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


def _own_beam(s):
    jk, st = _jk(), torch.cuda.current_stream().cuda_stream
    jk.dev_beam_select(s["args"], s["ws"], stream=st)
    jk.dev_paged_reorder(s["paged"], s["parents"], s["case"]["width"], s["status"], s["lens_out"], s["table_out"],
                         stream=st)
    return s["scores_out"], s["parents"], s["tokens"], s["done_out"], s["lens_out"], s["table_out"]


_own = {"tables": _own_tables, "append": _own_append, "attn": _own_attn, "beam": _own_beam}


def _plain_tables(s):
    """The plan by prefix sums: pages from the top of the free stack, request by request."""
    page, lens, new, table = s["case"]["page"], s["lens"], s["new"], s["table"]
    q_start = torch.zeros_like(s["q_start"])
    q_start[1:] = torch.cumsum(new, 0)
    have, need = _pages_of(lens, page), _pages_of(lens + new, page)
    more = need - have
    before = torch.cumsum(more, 0) - more
    j = torch.arange(table.shape[1], device=DEV, dtype=torch.int32)[None]
    fresh = (j >= have[:, None]) & (j < need[:, None])
    at = s["n_free"] - 1 - (before[:, None] + j - have[:, None])
    table.copy_(torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1).long()], table))
    t = torch.arange(s["cap"], device=DEV, dtype=torch.int32)
    of = (torch.searchsorted(q_start, t, right=True) - 1).to(torch.int32)
    live = t < q_start[-1]
    r = of.clamp(max=lens.numel() - 1).long()
    pos = t - q_start[r] + lens[r]
    cell = torch.where(live, pos, 0)
    slots = table[r, torch.div(cell, page, rounding_mode="floor").long()] * page + cell % page
    none = torch.full_like(t, -1)
    return (q_start, torch.where(live, slots, none), torch.where(live, pos, none), torch.where(live, of, none), table,
            lens + new, s["n_free"] - more.sum().to(torch.int32), torch.zeros_like(s["status"]))


def _plain_store(x, codes, scale, slots, page):
    """Quantizes x into its pages: a page's scale grows to its largest value, its older codes with it."""
    x = x.float()
    x = torch.where(torch.isfinite(x), x, 0.0)
    at, row = torch.div(slots, page, rounding_mode="floor").long(), (slots % page).long()
    top = torch.zeros_like(scale).index_reduce_(0, at, x.abs().amax(2), "amax")
    old = scale.clone()
    old[at[row == 0]] = 0.0
    # (a tensor of 127: by a number torch multiplies with the reciprocal on the GPU, which misses 4% of the quotients)
    d = torch.maximum(old, torch.where(top < TINY, 0.0, top / torch.full_like(top, 127.0)))
    touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=DEV)
    touched[at] = True
    hit = touched.nonzero()[:, 0]
    ratio = torch.where(d[hit] > 0, old[hit] / d[hit], 0.0)[..., None, None]
    codes[hit] = torch.round(codes[hit].float() * ratio).to(torch.int8)
    scale[hit] = d[hit]
    inv = torch.where(d > 0, 1.0 / d, 0.0)[at][..., None]
    codes[at, :, row] = torch.round(x * inv).clamp(-127, 127).to(torch.int8)


def _plain_append(s):
    page, read = s["case"]["page"], s["read"]
    _plain_store(s["k"], s["codes_k"], s["scale_k"], s["slots"], page)
    _plain_store(s["v"], s["codes_v"], s["scale_v"], s["slots"], page)
    at, row = torch.div(read, page, rounding_mode="floor").long(), (read % page).long()
    k = s["codes_k"][at, :, row].float() * s["scale_k"][at][..., None]
    v = s["codes_v"][at, :, row].float() * s["scale_v"][at][..., None]
    return s["scale_k"], s["scale_v"], k, v


def _plain_attn(s):
    """Softmax attention over the gathered cache, the requests padded to the longest."""
    case, q, q_start, lens = s["case"], s["q"], s["q_start"], s["lens"]
    b, kv, hd, page = lens.numel(), case["kv_heads"], case["head_dim"], case["page"]
    grp = case["heads"] // kv
    n_pages = -(-s["max_len"] // page)
    pages = s["table"][:, :n_pages].clamp(min=0).long()

    def gathered(codes, scale):
        x = codes[pages].float() * scale[pages][..., None, None]  # [b, pages, kv, page, hd]
        return x.transpose(1, 2).reshape(b, kv, n_pages * page, hd)

    t = torch.arange(q.shape[0], device=DEV)
    r = torch.searchsorted(q_start.long(), t, right=True) - 1
    i = t - q_start[r]
    x = torch.zeros((b, s["max_new"], case["heads"], hd), device=DEV)
    x[r, i] = q.float()
    x = x.reshape(b, -1, kv, grp, hd).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, hd)
    scores = torch.matmul(x, gathered(s["codes_k"], s["scale_k"]).transpose(2, 3).contiguous()) * hd ** -0.5
    scores = scores.view(b, kv, grp, s["max_new"], -1)
    pos = (lens - (q_start[1:] - q_start[:-1]))[:, None] + torch.arange(s["max_new"], device=DEV)[None]
    j = torch.arange(n_pages * page, device=DEV)
    seen = (j <= pos[..., None]) & (j < lens[:, None, None])
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    y = torch.matmul(p.view(b, kv, grp * s["max_new"], -1), gathered(s["codes_v"], s["scale_v"]))
    y = y.view(b, kv, grp, s["max_new"], hd).permute(0, 3, 1, 2, 4).reshape(b, s["max_new"], case["heads"], hd)
    return y[r, i].to(q.dtype)


def _plain_beam(s):
    """Totals of every continuation; a beam's own rank by logit, the group's by total, ties to the lowest index."""
    case = s["case"]
    g, w, v, page = case["groups"], case["width"], case["vocab"], case["page"]
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(1, keepdim=True)
    x, tok = torch.sort(x, dim=1, descending=True, stable=True)
    total = s["scores"].view(-1, 1) + ((x - top) - torch.log(torch.exp(x - top).sum(1, keepdim=True)))
    total, tok = total[:, :w], tok[:, :w]
    total = torch.where(torch.isnan(total), -math.inf, total)
    ended = (s["done"].view(-1, 1) != 0)
    first = torch.arange(min(w, v), device=DEV)[None] == 0
    # a finished hypothesis goes on as itself alone
    total = torch.where(ended, torch.where(first, s["scores"].view(-1, 1), -math.inf), total).view(g, -1)
    tok = torch.where(ended, s["eos"], tok).view(g, -1)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)
    best, at = best[:, :w].contiguous(), at[:, :w]
    parents, tokens = (at // min(w, v)).to(torch.int32), tok.gather(1, at).to(torch.int32)
    done = ((s["done"].gather(1, parents.long()) != 0) | (tokens == s["eos"])).to(torch.int32)
    # the cache rows: full pages are the parent's, the open one is the row's own
    rows = (torch.arange(g, device=DEV)[:, None] * w + parents).view(-1).long()
    lens = s["lens"][rows]
    j = torch.arange(s["table"].shape[1], device=DEV)[None]
    full = torch.div(lens, page, rounding_mode="floor")[:, None]
    mine = (j == full) & ((lens % page) != 0)[:, None]
    table = torch.where(j < full, s["table"][rows], torch.where(mine, s["owned"], -1))
    return best, parents, tokens, done, lens, table


_plain = {"tables": _plain_tables, "append": _plain_append, "attn": _plain_attn, "beam": _plain_beam}


# ------------------------------------------------------------------ what a pass needs, and its values in 64 bits
def _mean(case):
    """Mean length held and number of new tokens of a case's requests."""
    if case["kind"] == "attn":
        n = case["new"] * (2 / 3 if case["ragged"] and case["new"] > 16 else 1)
        return case["held"] * (9 / 16 if case["ragged"] else 1), n
    return case["held"] / 2, case["prompt"] / 2 if case["prompt"] else 6 / 7


def work(case):
    if case["kind"] == "beam":
        rows = case["groups"] * case["width"]
        es = 4 if case["dtype"] == "f32" else 2
        table = rows * (2 / 3 * case["held"] / case["page"]) * 8
        return {"bytes": rows * (case["vocab"] * es + 32) + table, "flops": 4 * rows * case["vocab"]}
    held, new = _mean(case)
    tokens = case["requests"] * new
    if case["kind"] == "tables":
        return {"bytes": 12 * tokens + 8 * tokens / case["page"] + 16 * case["requests"], "flops": 4 * tokens}
    kv, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    es = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "append":
        back = case["requests"] * (new + page / 2)  # the tokens read back, as codes and as values
        return {"bytes": 2 * kv * hd * (tokens * (es + 1) + back * 5), "flops": 2 * kv * hd * (4 * tokens + back)}
    seen, whole = held + new / 2, held + new
    if case["window"]:
        seen, whole = min(seen, case["window"]), min(whole, case["window"] + new)
    cache = case["requests"] * whole * kv * 2 * (hd + 4 / page)
    return {"bytes": cache + 2 * tokens * case["heads"] * hd * es, "flops": 4 * tokens * seen * case["heads"] * hd}


def exact(case, seed):
    with torch.no_grad():
        return {"append": _exact_append, "attn": _exact_attn, "beam": _exact_beam}.get(case["kind"], lambda *a: None)(
            case, prepare(case, seed))


def _exact_append(case, s):
    """Page by page from the definition: x / (largest / 127), rounded, times that scale again."""
    out, page = [], case["page"]
    n_pages, kv = s["scale_k"].shape
    slots, read = s["slots"].long(), s["read"].long()
    for x, codes, scale in ((s["k"], s["codes_k"], s["scale_k"]), (s["v"], s["codes_v"], s["scale_v"])):
        x, held = x.double(), scale.double()
        held.view(-1, kv)[slots[slots % page == 0] // page] = 0
        peak = torch.zeros((n_pages, kv), dtype=torch.float64, device=DEV)
        peak.scatter_reduce_(0, (slots // page)[:, None].expand(-1, kv), x.abs().amax(-1), "amax")
        d = torch.maximum(held, peak / 127)
        whole = codes.double().transpose(1, 2).reshape(n_pages * page, kv, -1)
        per_slot = lambda y: y.repeat_interleave(page, 0)[:, :, None]  # noqa: E731
        # (pages that the step does not write to keep their scale: peak is 0 there)
        whole = torch.round(whole * per_slot(held) / per_slot(d))
        whole[slots] = torch.round(x / d[slots // page][..., None])
        out.append((d, whole[read] * d[read // page][..., None]))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attn(case, s):
    page, kv, hd = case["page"], case["kv_heads"], case["head_dim"]
    grp = case["heads"] // kv
    y = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    starts, lens = s["q_start"].tolist(), s["lens"].tolist()
    for r, n in enumerate(lens):
        pages = s["table"][r, :-(-n // page)].long()
        i0, i1 = starts[r], starts[r + 1]
        pos = torch.arange(n - (i1 - i0), n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)[None]
        unseen = (j > pos) | ((j <= pos - case["window"]) if case["window"] else False)
        for h in range(kv):
            k = (s["codes_k"][pages, h].double() * s["scale_k"][pages, h, None, None].double()).view(-1, hd)[:n]
            v = (s["codes_v"][pages, h].double() * s["scale_v"][pages, h, None, None].double()).view(-1, hd)[:n]
            for e in range(h * grp, (h + 1) * grp):
                a = (s["q"][i0:i1, e].double() @ k.T) / math.sqrt(hd)
                y[i0:i1, e] = torch.softmax(a.masked_fill(unseen, -math.inf), -1) @ v
    return y


def _exact_beam(case, s):
    g, w = case["groups"], case["width"]
    logp = torch.log_softmax(s["logits"].double(), -1).view(g, w, -1)
    total = s["scores"].double()[..., None] + logp
    ended = s["done"] != 0
    total[ended] = -math.inf
    total[..., 0] = torch.where(ended, s["scores"].double(), total[..., 0])
    return torch.topk(total.view(g, -1), w, 1)[0], None, None, None, None, None
