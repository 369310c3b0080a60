"""Beam search's selection on the GPU against a plain implementation in 64 bits.

Parents and tokens are compared exactly (random totals lie far enough apart; ties are made of equal inputs). A total
sums score, x - m and log(sum): its f32 value is off by at most 2^-22 of |score| + |x - m| + |log sum| for the roundings, plus
the sum's own relative error, (vocab / 64 + 64) 2^-24 for its additions and 2^-21 for its exponentials.
"""
import numpy as np
import pytest

import jk
import paged_ref as R

pytestmark = pytest.mark.gpu


def run(torch, logits, scores, done, eos, ends=True, stride=None, at=0):
    groups, width = scores.shape
    x = logits.cuda()
    if stride:
        buf = torch.full((x.shape[0] * stride + at + 8,), 100.0, dtype=x.dtype, device="cuda")  # (never to be chosen)
        y = torch.as_strided(buf, x.shape, (stride, 1), at)
        y.copy_(x)
        x = y
    ints = lambda: torch.full((groups, width), -7, dtype=torch.int32, device="cuda")  # noqa: E731
    out = [torch.full((groups, width), float("nan"), device="cuda"), ints(), ints(), ints() if ends else None]
    dn = None if done is None else torch.tensor(done, dtype=torch.int32).cuda()
    a = jk.beam_args(x, torch.tensor(scores, dtype=torch.float32).cuda(), dn, *out[:3], out[3], eos=eos)
    ws = torch.full((jk.beam_workspace_bytes(a),), 0xFF, dtype=torch.uint8, device="cuda")
    jk.dev_beam_select(a, ws)
    torch.cuda.synchronize()
    return [None if o is None else o.cpu().numpy() for o in out]


def check(torch, logits, scores, done=None, eos=-1, **kw):
    got = run(torch, logits, scores, done, eos, **kw)
    groups, width = scores.shape
    x = logits.float().numpy().reshape(groups, width, -1)
    for g in range(groups):
        total, parent, token = R.beam(x[g], scores[g].astype(np.float32), None if done is None else done[g], eos)
        assert got[1][g].tolist() == parent and got[2][g].tolist() == token, g
        for t, w in zip(got[0][g], total):
            assert t == w or abs(t - w) <= (abs(scores).max() + abs(w) + 40) * 2.0 ** -22 + (x.shape[2] / 64 + 64) * 2.0 ** -24 + 2.0 ** -21
        if got[3] is not None:
            ended = [int((done is not None and done[g][p] != 0) or t == eos) for p, t in zip(parent, token)]
            assert got[3][g].tolist() == ended
    return got


def inputs(torch, groups, width, vocab, dtype, seed):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((groups * width, vocab)).astype(np.float32) * 3
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    return torch.from_numpy(x).to(t), -np.sort(rng.random((groups, width)).astype(np.float32) * 4)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("groups,width,vocab", [(1, 1, 1), (1, 4, 3), (2, 3, 64), (3, 5, 2047), (1, 8, 2048), (2, 2, 2049),
                                                (2, 32, 4999), (1, 4, 32000), (1, 3, 140001)])
def test_select(gpu, dtype, groups, width, vocab):
    x, scores = inputs(gpu, groups, width, vocab, dtype, vocab + width)
    check(gpu, x, scores)
    done = np.random.default_rng(width).integers(0, 3, scores.shape) == 0
    check(gpu, x, scores, done.astype(np.int32), eos=vocab - 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width", [1, 4, 8, 32])
def test_ties_go_to_the_lowest(gpu, dtype, width):
    """Rows of few different values, equal rows with equal scores, and rows of one value: order by hypothesis and token."""
    torch = gpu
    rng = np.random.default_rng(width)
    x = torch.from_numpy(rng.integers(-2, 3, (2 * width, 5000)).astype(np.float32)).to(
        {"f32": torch.float32, "bf16": torch.bfloat16}[dtype])
    scores = np.full((2, width), -1.5, np.float32)
    # (totals of different rows that are equal but for rounding are no ties to compare: every row of a group is the same)
    x = x.view(2, width, -1)[:, :1].expand(2, width, 5000).reshape(2 * width, 5000).contiguous()
    check(torch, x, scores)
    check(torch, torch.zeros_like(x), scores)
    z = torch.zeros_like(x)
    z[:, 1::2] = -0.0  # (equal to 0)
    check(torch, z, scores)


def test_masked_logits(gpu):
    """-inf, NaN and +inf logits, rows with nothing left, scores of -inf: what is left is chosen, in order."""
    torch = gpu
    x, scores = inputs(torch, 2, 4, 3001, "f32", 7)
    x[0] = float("-inf")
    x[1, 5:] = float("-inf")
    x[2, ::2] = float("nan")
    x[3, 10] = float("inf")
    x[4:, :] = float("-inf")
    x[5, 2999] = 1.0
    check(torch, x, scores)
    scores[0, 1:] = -np.inf  # the first step: one hypothesis is there
    x, _ = inputs(torch, 2, 4, 3001, "f32", 8)
    got = check(torch, x, scores)
    assert got[1][0].tolist() == [0] * 4
    x.fill_(float("nan"))
    check(torch, x, scores)


def test_finished_hypotheses(gpu):
    torch = gpu
    x, scores = inputs(torch, 1, 4, 500, "f32", 9)
    got = check(torch, x, scores, np.ones((1, 4), np.int32), eos=3)
    assert got[1][0].tolist() == [0, 1, 2, 3] and np.array_equal(got[0][0], scores[0])
    x[:, 3] = 50  # everybody finishes now
    got = check(torch, x, scores, np.zeros((1, 4), np.int32), eos=3)
    assert got[3].all()
    check(torch, x, scores, None, eos=3)
    check(torch, x, scores, None, eos=-1, ends=False)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_strided_and_unaligned_rows(gpu, dtype):
    x, scores = inputs(gpu, 2, 3, 4100, dtype, 10)
    for stride, at in ((4104, 0), (4101, 0), (4104, 1), (5000, 8)):
        check(gpu, x, scores, stride=stride, at=at)
