"""Arguments that the paged cache's operators refuse, checked before any device work (so no GPU is needed)."""
import ctypes as C

import pytest

import jk

P = 0x10000  # an address that no call gets as far as using


def paged(**kw):
    f = dict(n_requests=4, max_pages=8, n_pages=32, page=16, lens=P, table=P, owned=2 * P, free_pages=P, n_free=P)
    f.update(kw)
    return jk.PagedC(**f)


def cache(**kw):
    f = dict(n_pages=32, page=16, n_kv=2, head_dim=64, k=P, v=P, k_scale=P, v_scale=P)
    f.update(kw)
    return jk.KvQ8C(**f)


def step(**kw):
    f = dict(max_tokens=8, q_start=P, slots=P, positions=P, requests=P, status=P)
    f.update(kw)
    return jk.PagedStepC(**f)


def attn(**kw):
    f = dict(q=P, out=P, dtype=jk.F32, n_tokens=4, n_heads=8, n_requests=4, max_pages=8, q_start=P, lens=P, table=P,
             max_new=1, max_len=100, scale=0.125, window=0)
    f.update(kw)
    return jk.AttnQ8ArgsC(**f)


def beam(**kw):
    f = dict(logits=P, dtype=jk.F32, groups=1, width=4, vocab=1000, stride=0, scores=P, done=2 * P, eos=2,
             scores_out=3 * P, parents=4 * P, tokens=5 * P, done_out=6 * P)
    f.update(kw)
    return jk.BeamArgsC(**f)


def refused(kind, match, fn, *args):
    with pytest.raises(kind, match=match):
        fn(*args)


TB, CM = jk.TensorBoundsError, jk.CapabilityMismatch


@pytest.mark.parametrize("kw,match", [
    ({"lens": None}, "null array"), ({"owned": None}, "null array"), ({"page": 24}, "tokens a page"),
    ({"page": 8}, "tokens a page"), ({"page": 512}, "tokens a page"), ({"n_requests": 0}, "no requests"),
    ({"max_pages": 0}, "no requests"), ({"n_pages": 2 ** 27}, "int32"), ({"max_pages": 2 ** 28}, "int32")])
def test_pages(kw, match):
    p = paged(**kw)
    refused(TB, match, jk.dev_paged_reset, p)
    refused(TB, match, jk.dev_paged_extend, p, P, step())
    refused(TB, match, jk.dev_paged_release, p, P)
    refused(TB, match, jk.dev_paged_reorder, p, P, 2, P)
    refused(TB, match, lambda: jk.dev_kv_reorder_q8(cache(), p, P, 2, P))


def test_steps_and_reorderings():
    p = paged()
    refused(TB, "null counts", jk.dev_paged_extend, p, None, step())
    refused(TB, "null counts", jk.dev_paged_extend, p, P, step(status=None))
    refused(TB, "null slots", jk.dev_paged_extend, p, P, step(slots=None))
    refused(TB, "int32", jk.dev_paged_extend, p, P, step(max_tokens=2 ** 31))
    refused(TB, "null flags", jk.dev_paged_release, p, None)
    for width in (0, 3, 33):
        refused(TB, "width", jk.dev_paged_reorder, p, P, width, P)
        refused(TB, "width", lambda: jk.dev_kv_reorder_q8(cache(), p, P, width, P))
    refused(TB, "same array", jk.dev_paged_reorder, paged(owned=P), P, 2, P)
    refused(TB, "both or neither", jk.dev_paged_reorder, p, P, 2, P, P, None)
    refused(TB, "is owned", jk.dev_paged_reorder, p, P, 2, P, P, 2 * P)
    refused(TB, "null parents", jk.dev_paged_reorder, p, None, 2, P)
    refused(TB, "null parents", jk.dev_paged_reorder, p, P, 2, None)
    refused(TB, "for tables of", lambda: jk.dev_kv_reorder_q8(cache(page=32), p, P, 2, P))
    refused(TB, "for tables of", lambda: jk.dev_kv_reorder_q8(cache(n_pages=31), p, P, 2, P))


def append(c, k=P, v=P, dtype=jk.F32, n=4, slots=P):
    jk._check(jk.lib().jk_kv_append_q8(None, C.byref(c), C.c_void_p(k), C.c_void_p(v), dtype, C.c_size_t(n), C.c_size_t(0),
                                       C.c_size_t(0), C.c_void_p(slots)))


def read(c, slots=P, n=4, dtype=jk.F32, k=P, v=P):
    jk._check(jk.lib().jk_kv_read_q8(None, C.byref(c), C.c_void_p(slots), C.c_size_t(n), dtype, C.c_void_p(k),
                                     C.c_void_p(v)))


@pytest.mark.parametrize("kw,kind,match", [
    ({"k": None}, TB, "null array"), ({"v_scale": None}, TB, "null array"), ({"k": P + 8}, TB, "aligned"),
    ({"page": 48}, TB, "tokens a page"), ({"head_dim": 0}, CM, "head dimension"), ({"head_dim": 72}, CM, "head dimension"),
    ({"head_dim": 272}, CM, "head dimension"), ({"n_kv": 0}, TB, "kv heads"), ({"n_pages": 0}, TB, "int32"),
    ({"n_pages": 2 ** 27}, TB, "int32")])
def test_caches(kw, kind, match):
    c = cache(**kw)
    refused(kind, match, append, c)
    refused(kind, match, read, c)
    refused(kind, match, lambda: jk.dev_attn_q8(c, attn()))
    refused(kind, match, lambda: jk.dev_kv_reorder_q8(c, paged(), P, 2, P))


def test_appending_and_reading():
    c = cache()
    refused(CM, "element type", lambda: append(c, dtype=2))
    refused(TB, "null keys", lambda: append(c, k=None))
    refused(TB, "null keys", lambda: append(c, slots=None))
    refused(TB, "aligned to their elements", lambda: append(c, v=P + 2))
    refused(TB, "too many", lambda: append(c, n=2 ** 28))
    refused(CM, "element type", lambda: read(c, dtype=-1))
    refused(TB, "null slots", lambda: read(c, slots=None))
    refused(TB, "aligned to their elements", lambda: read(c, k=P + 1))
    refused(TB, "too many", lambda: read(c, n=2 ** 30))
    append(c, n=0)  # nothing to do is no error
    read(c, n=0)


@pytest.mark.parametrize("kw,kind,match", [
    ({"dtype": 7}, CM, "element type"), ({"n_heads": 7}, TB, "query heads"), ({"n_heads": 0}, TB, "query heads"),
    ({"n_requests": 0}, TB, "requests"), ({"max_pages": 0}, TB, "requests"), ({"n_tokens": 2 ** 30}, TB, "int32"),
    ({"q": None}, TB, "null"), ({"table": None}, TB, "null"), ({"q": P + 2}, TB, "aligned"),
    ({"scale": float("nan")}, TB, "scale"), ({"scale": float("inf")}, TB, "scale"),
    ({"n_requests": 2 ** 24, "max_new": 4}, TB, "too many"),
    ({"n_requests": 1, "max_len": 100000, "max_pages": 10000}, TB, "workspace")])
def test_attention(kw, kind, match):
    refused(kind, match, lambda: jk.dev_attn_q8(cache(), attn(**kw)))


def test_attention_of_nothing():
    jk.dev_attn_q8(cache(), attn(n_tokens=0))
    jk.dev_attn_q8(cache(), attn(max_new=0))
    assert jk.attn_q8_workspace_bytes(cache(), attn(n_heads=7)) == 0


@pytest.mark.parametrize("kw,kind,match", [
    ({"dtype": 3}, CM, "element type"), ({"width": 0}, TB, "width"), ({"width": 33}, TB, "width"),
    ({"vocab": 0}, CM, "logits a row"), ({"vocab": 2 ** 20 + 1}, CM, "logits a row"), ({"groups": 0}, TB, "groups"),
    ({"groups": 70000}, TB, "groups"), ({"stride": 999}, TB, "stride"), ({"logits": None}, TB, "null"),
    ({"tokens": None}, TB, "null"), ({"eos": -1}, TB, "does not finish"), ({"eos": 1000}, TB, "does not finish"),
    ({"scores_out": P}, TB, "computed from"), ({"done_out": 2 * P}, TB, "computed from"), ({"logits": P + 2}, TB, "aligned"),
    ({}, TB, "workspace")])
def test_beam(kw, kind, match):
    refused(kind, match, lambda: jk.dev_beam_select(beam(**kw), None))


def test_beam_workspace():
    need = jk.beam_workspace_bytes(beam())
    assert need > 0 and jk.beam_workspace_bytes(beam(width=0)) == 0
    a = beam()
    for ws, n in ((P, need - 1), (P + 8, need)):
        with pytest.raises(TB, match="workspace"):
            jk._check(jk.lib().jk_beam_select(None, C.byref(a), C.c_void_p(ws), C.c_size_t(n)))
