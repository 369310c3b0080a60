"""What the Python layer of the paged cache's operators refuses before a call (torch tensors on the CPU: no GPU needed)."""
import pytest
import torch

import jk

TB = jk.TensorBoundsError


def cache(pages=4, kv=2, page=16, hd=64):
    codes = [torch.zeros((pages, kv, page, hd), dtype=torch.int8) for _ in range(2)]
    return codes + [torch.zeros((pages, kv)) for _ in range(2)]


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_caches():
    k, v, ks, vs = cache()
    c = jk.kv_q8(k, v, ks, vs)
    assert (c.n_pages, c.n_kv, c.page, c.head_dim) == (4, 2, 16, 64) and c.tensors[0] is k
    for bad in ((k[:3], v, ks, vs), (k.float(), v, ks, vs), (k, v, ks[:3], vs), (k, v, ks, vs.double()),
                (k.transpose(1, 2), v, ks, vs)):
        with pytest.raises(TB):
            jk.kv_q8(*bad)


def test_appending():
    c = jk.kv_q8(*cache())
    x = torch.zeros((5, 2, 64))
    for k, v, slots in ((x, x[:4], ints(5)), (x, x.half(), ints(5)), (x, x, ints(4)), (x, x, ints(5).long()),
                        (x[:, :1], x[:, :1], ints(5)), (x.transpose(1, 2), x.transpose(1, 2), ints(5)),
                        (x, x.transpose(0, 1).contiguous().transpose(0, 1), ints(5)), (x[0], x[0], ints(2))):
        with pytest.raises(TB):
            jk.dev_kv_append_q8(c, k, v, slots)
    with pytest.raises(jk.CapabilityMismatch):
        jk.dev_kv_append_q8(c, x.double(), x.double(), ints(5))
    with pytest.raises(TB):
        jk.dev_kv_read_q8(c, ints(5), torch.zeros((4, 2, 64)), None)
    with pytest.raises(TB):
        jk.dev_kv_read_q8(c, ints(5), x, x.half())


def test_strides_of_single_tokens():
    x = torch.zeros((7, 2, 64))
    assert jk._strides(x) == (128, 64) and jk._strides(x[:1]) == (0, 64) and jk._strides(x[:1, :1]) == (0, 0)
    assert jk._strides(torch.as_strided(x, (1, 1, 64), (999, 5, 1))) == (0, 0)


def test_expanded_tensors():
    """A stride of 0 means packed to the library: a tensor that repeats one row must not reach it as one."""
    c = jk.kv_q8(*cache())
    for x in (torch.zeros((1, 2, 64)).expand(5, 2, 64), torch.zeros((5, 1, 64)).expand(5, 2, 64)):
        with pytest.raises(TB, match="expanded"):
            jk.dev_kv_append_q8(c, x, x, ints(5))
        with pytest.raises(TB, match="expanded"):
            jk.attn_q8_args(x, torch.zeros((5, 2, 64)), ints(3), ints(2), ints(2, 8), 1, 10, 0.125)
    s = torch.zeros((2, 3))
    with pytest.raises(TB, match="expanded"):
        jk.beam_args(torch.zeros((1, 100)).expand(6, 100), s, ints(2, 3), s.clone(), ints(2, 3), ints(2, 3), ints(2, 3))


def test_attention_arguments():
    q = torch.zeros((5, 4, 64))
    good = [q, torch.zeros_like(q), ints(3), ints(2), ints(2, 8)]
    a = jk.attn_q8_args(*good, 1, 10, 0.125)
    assert (a.n_tokens, a.n_heads, a.n_requests, a.max_pages, a.window) == (5, 4, 2, 8, 0)
    for i, bad in ((1, torch.zeros((4, 4, 64))), (1, q.half()), (2, ints(2)), (3, ints(3)), (4, ints(8)), (4, ints(3, 8)),
                   (2, ints(3).long()), (0, q.transpose(1, 2))):
        args = list(good)
        args[i] = bad
        with pytest.raises(TB):
            jk.attn_q8_args(*args, 1, 10, 0.125)


def test_beam_and_page_arguments():
    x, s = torch.zeros((6, 100)), torch.zeros((2, 3))
    good = [x, s, ints(2, 3), s.clone(), ints(2, 3), ints(2, 3), ints(2, 3)]
    a = jk.beam_args(*good, eos=2)
    assert (a.groups, a.width, a.vocab, a.stride) == (2, 3, 100, 100)
    assert jk.beam_args(torch.zeros((6, 200))[:, :100], *good[1:]).stride == 200
    for i, bad in ((0, torch.zeros((5, 100))), (0, torch.zeros((100, 6)).T), (2, ints(3, 2)), (3, s.double()), (4, ints(2, 2)),
                   (5, ints(2, 3).long())):
        args = list(good)
        args[i] = bad
        with pytest.raises(TB):
            jk.beam_args(*args)
    with pytest.raises(TB):
        jk.paged(ints(2), ints(3, 8), ints(3, 8), ints(9), ints(1), 16)
    with pytest.raises(TB):
        jk.paged_step(ints(3), ints(4), ints(5), ints(4), ints(1))


def test_tables_and_flags_of_the_wrong_size_or_type():
    """Counts, flags and parents are read one a request: the usual int64 tensor or a short one must not get that far."""
    p = jk.paged(ints(6), ints(6, 8), ints(6, 8), ints(40), ints(1), 16)
    step = jk.paged_step(ints(7), ints(9), ints(9), ints(9), ints(1))
    calls = [lambda: jk.paged(ints(6), ints(6, 8), ints(6, 8), ints(40), ints(0), 16),
             lambda: jk.paged_step(ints(7), ints(9), ints(9), ints(9), ints(2)),
             lambda: jk.dev_paged_extend(p, ints(6), jk.paged_step(ints(6), ints(9), ints(9), ints(9), ints(1))),
             lambda: jk.dev_paged_extend(p, ints(6), step, ints(5), ints(1)),
             lambda: jk.dev_paged_extend(p, ints(6), step, ints(6), ints(1).long()),
             lambda: jk.dev_paged_reorder(p, ints(2, 3), 3, ints(1).long()),
             lambda: jk.dev_paged_reorder(p, ints(2, 3), 3, ints(1), ints(6), ints(6, 7)),
             lambda: jk.dev_kv_reorder_q8(jk.kv_q8(*cache(40)), p, ints(2, 3), 3, ints(0))]
    for x in (ints(5), ints(6).long(), ints(6, 2)[:, 0]):
        calls += [lambda x=x: jk.dev_paged_extend(p, x, step), lambda x=x: jk.dev_paged_release(p, x),
                  lambda x=x: jk.dev_paged_reorder(p, x, 3, ints(1)),
                  lambda x=x: jk.dev_kv_reorder_q8(jk.kv_q8(*cache(40)), p, x, 3, ints(1))]
    for call in calls:
        with pytest.raises(TB):
            call()


def test_queries_of_another_head_dimension():
    q = torch.zeros((5, 4, 80))
    a = jk.attn_q8_args(q, torch.zeros_like(q), ints(3), ints(2), ints(2, 8), 1, 10, 0.125)
    with pytest.raises(TB, match="80 channels"):
        jk.dev_attn_q8(jk.kv_q8(*cache()), a)
