"""Sizes at which the attention's 32-bit token numbers would end, refused before any device work (no GPU needed)."""
import pytest

import jk

P = 0x10000  # an address that no call gets as far as using


@pytest.mark.parametrize("page", [16, 64, 256])
def test_tables_of_almost_2_to_the_31_tokens(page):
    """The kernels look some hundred tokens past a request's end for what to load next."""
    c = jk.KvQ8C(n_pages=32, page=page, n_kv=2, head_dim=64, k=P, v=P, k_scale=P, v_scale=P)

    def call(max_pages):
        jk.dev_attn_q8(c, jk.AttnQ8ArgsC(q=P, out=P, dtype=jk.F32, n_tokens=4, n_heads=8, n_requests=4, max_pages=max_pages,
                                         q_start=P, lens=P, table=P, max_new=1, max_len=10 ** 6, scale=0.125, window=0))
    for max_pages in ((2 ** 31 - 1) // page, (2 ** 31 - 4096) // page + 1):
        with pytest.raises(jk.TensorBoundsError, match="requests of"):
            call(max_pages)
    with pytest.raises(jk.TensorBoundsError, match="workspace"):
        call((2 ** 31 - 4096) // page)  # (as far as the next check)
