"""Edges of the e4m3 operators: memory that was never written, weights far below a row's
largest, tables with pages that are none. Against numpy in 64 bits (fp8_oracle).
"""
import numpy as np
import pytest

import fp8_oracle as O
import test_fp8_operators as F

I32 = np.int32


# ---- GPU: memory that was never written --------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dh,batch,kv,nq,n,gone", [
    # two tiles a workgroup, two halves of the pages: odd numbers of pages, and one alone
    (64, 1, 1, 40, 700, False), (128, 1, 1, 40, 700, False), (256, 1, 1, 40, 700, False),
    (64, 3, 2, 33, 60, False), (128, 3, 2, 33, 60, False), (256, 3, 2, 33, 60, False),
    # four tiles a workgroup, and a page of the table that is none
    (64, 97, 8, 17, 150, True), (128, 97, 8, 17, 150, True), (256, 17, 8, 32, 150, True),
    # few columns
    (128, 3, 2, 1, 700, True), (256, 2, 1, 3, 200, True)])
def test_attention_beside_bytes_never_written(gpu_ctx, dh, batch, kv, nq, n, gone):
    """Page 0 belongs to nobody, and every byte that was never written is 0xFF: NaN as a code and
    as a scale. A page that is none, in the table or behind a range's last, takes no scale
    from there."""
    rng = np.random.default_rng(dh + n)
    blocks = -(-n // 64)
    table = (1 + rng.permutation(batch * blocks).reshape(batch, blocks)).astype(I32)
    c = O.Cache(1 + batch * blocks, kv, dh, fill=0xFF)
    c.k_exp[:], c.v_exp[:] = 255, 255
    cu = np.arange(batch + 1, dtype=I32) * n
    at = np.concatenate([table[b, np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64
                         for b in range(batch)])
    k, v = rng.standard_normal((2, batch * n, kv, dh))
    c.append(k, v, cu, at)
    assert (c.v_exp[0] == 255).all() and (c.v_exp[1:] != 255).all()
    qcu, lens = np.arange(batch + 1, dtype=I32) * nq, np.full(batch, n, I32)
    q = rng.standard_normal((batch * nq, 2 * kv, dh))
    scale = dh ** -0.5
    want, val = F.attend(gpu_ctx, c, q, "bf16", table, qcu, lens, scale, False, 0, False)
    F.check_attention(c, want, val, table, qcu, lens, scale, False, 0, "bf16", False)
    if gone:  # the first block of the last request: its other keys alone
        bad = table.copy()
        bad[-1, 0] = -1
        got, _ = F.attend(gpu_ctx, c, q, "bf16", bad, qcu, lens, scale, False, 0, False)
        assert np.array_equal(got[:-nq], want[:-nq])
        F.check_attention(c, got[-nq:], val[-nq:], table[-1:, 1:], np.array([0, nq], I32),
                          lens[-1:] - 64, scale, False, 0, "bf16", False)
