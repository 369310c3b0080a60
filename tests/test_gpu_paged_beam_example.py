"""The serving operators together: examples/paged_beam_search.py on the GPU, step by step.

Every selection is compared with the plain implementation on the same logits, and across every reordering each row has to hold
exactly the keys and values that the row it goes on from held (codes and scales are moved, never changed).
"""
import importlib.util
import os

import numpy as np
import pytest

import jk
import paged_ref as R

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_beam_search.py")


@pytest.fixture(scope="module")
def example(gpu):
    spec = importlib.util.spec_from_file_location("paged_beam_search", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def contents(torch, batch, cache, page=16):
    """Each row's keys and values, read back by its table."""
    lens, table = batch.lens.tolist(), batch.table
    out = []
    for r, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        slots = (table[r, t // page] * page + t % page).to(torch.int32)
        k = torch.empty((n, cache.n_kv, cache.head_dim), device="cuda")
        v = torch.empty_like(k)
        jk.dev_kv_read_q8(cache, slots, k, v)
        out.append((k, v))
    return out


@pytest.mark.parametrize("width,lengths", [(1, [5]), (4, [16, 3, 41]), (5, [15, 33])])
def test_search(gpu, example, width, lengths):
    torch = gpu
    model = example.Decoder()
    rng = np.random.default_rng(width)
    prompts = [rng.integers(3, model.vocab, n).tolist() for n in lengths]
    held, steps = {}, []

    def seen(event, **w):
        if event == "selected":
            x = w["logits"].cpu().numpy().reshape(len(lengths), width, -1)
            for g in range(len(lengths)):
                total, parent, token = R.beam(x[g], w["scores"][g].cpu().numpy(), w["done"][g].tolist(), w["eos"])
                assert w["parents"][g].tolist() == parent and w["chosen"][g].tolist() == token
                # (totals of a few hundred at most: f32 sums of three terms and a logarithm of 1000 exponentials)
                assert np.allclose(w["best"][g].cpu().numpy(), total, rtol=1e-6, atol=1e-4)
            steps.append(w["parents"].view(-1).tolist())
        elif event == "reordering":
            held["rows"] = [contents(torch, w["batch"], c) for c in w["caches"]]
        else:
            for before, cache in zip(held["rows"], w["caches"]):
                for r, (k, v) in enumerate(contents(torch, w["batch"], cache)):
                    k0, v0 = before[r // width * width + steps[-1][r]]
                    assert torch.equal(k, k0) and torch.equal(v, v0)

    scores, history = example.search(model, prompts, width, 20, seen=seen)
    assert history.shape == (len(lengths), width, 20) and len(steps) == 20
    assert torch.all(scores[:, :-1] >= scores[:, 1:]) and bool(torch.isfinite(scores).all())
    # hypotheses differ unless they ended
    for g in range(len(lengths)):
        rows = [tuple(h) for h in history[g].tolist()]
        assert len(set(rows)) == width


def test_search_on_another_stream(gpu, example):
    """The same search on a stream of its own gives the same hypotheses."""
    torch = gpu
    model = example.Decoder()
    prompts = [[5, 9, 200, 31], [77] * 20]
    want = example.search(model, prompts, 3, 6)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = example.search(model, prompts, 3, 6)
    torch.cuda.synchronize()
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
