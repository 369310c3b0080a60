"""Tensors in host memory do not reach the serving kernels: the Python layer refuses them at the call (no GPU needed)."""
import pytest
import torch

import jk


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def calls():
    p = jk.paged(ints(6), ints(6, 8), ints(6, 8), ints(40), ints(1), 16)
    step = jk.paged_step(ints(7), ints(9), ints(9), ints(9), ints(1))
    c = jk.kv_q8(*(torch.zeros((40, 2, 16, 64), dtype=torch.int8) for _ in range(2)), *(torch.zeros((40, 2)) for _ in range(2)))
    x = torch.zeros((5, 2, 64))
    q = torch.zeros((5, 4, 64))
    a = jk.attn_q8_args(q, torch.zeros_like(q), ints(7), ints(6), ints(6, 8), 1, 10, 0.125)
    s = torch.zeros((2, 3))
    b = jk.beam_args(torch.zeros((6, 100)), s, ints(2, 3), s.clone(), ints(2, 3), ints(2, 3), ints(2, 3), eos=2)
    P = 0x10000  # an address, taken as it is
    rp, rs = (jk.PagedC(6, 8, 40, 16, P, P, 2 * P, P, P), jk.PagedStepC(9, P, P, P, P, P))
    rc = jk.KvQ8C(40, 16, 2, 64, P, P, P, P)
    return {
        "reset": lambda: jk.dev_paged_reset(p),
        "extend": lambda: jk.dev_paged_extend(p, P, rs),
        "extend, step": lambda: jk.dev_paged_extend(rp, P, step),
        "extend, counts": lambda: jk.dev_paged_extend(rp, ints(6), rs),
        "extend, lengths": lambda: jk.dev_paged_extend(rp, P, rs, ints(6), ints(1)),
        "release": lambda: jk.dev_paged_release(p, P),
        "release, flags": lambda: jk.dev_paged_release(rp, ints(6)),
        "reorder": lambda: jk.dev_paged_reorder(p, P, 3, P),
        "reorder, parents": lambda: jk.dev_paged_reorder(rp, ints(2, 3), 3, P),
        "reorder, status": lambda: jk.dev_paged_reorder(rp, P, 3, ints(1)),
        "append": lambda: jk.dev_kv_append_q8(c, x, x, ints(5)),
        "append, keys": lambda: jk.dev_kv_append_q8(rc, x, x, P),
        "read": lambda: jk.dev_kv_read_q8(c, ints(5), x, None),
        "read, output": lambda: jk.dev_kv_read_q8(rc, ints(5), x, None),
        "move": lambda: jk.dev_kv_reorder_q8(c, rp, P, 3, P),
        "move, tables": lambda: jk.dev_kv_reorder_q8(rc, p, P, 3, P),
        "attention": lambda: jk.dev_attn_q8(rc, a),
        "attention, cache": lambda: jk.dev_attn_q8(c, jk.AttnQ8ArgsC(dtype=jk.F32, n_tokens=4, n_heads=8, n_requests=4)),
        "beam": lambda: jk.dev_beam_select(b, torch.zeros(1 << 20, dtype=torch.uint8)),
    }


@pytest.mark.parametrize("name", list(calls()))
def test_refused(name):
    with pytest.raises(jk.TensorBoundsError, match="host memory"):
        calls()[name]()


def test_workspaces():
    for call in (lambda ws: jk.dev_attn_q8(jk.KvQ8C(), jk.AttnQ8ArgsC(), ws), lambda ws: jk.dev_beam_select(jk.BeamArgsC(), ws)):
        with pytest.raises(jk.TensorBoundsError, match="host memory"):
            call(torch.zeros(1 << 20, dtype=torch.uint8))
