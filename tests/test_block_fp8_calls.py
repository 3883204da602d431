"""Host side of the block-scaled FP8 product's calls: strides that say nothing.  No launch, made-up addresses."""
from __future__ import annotations

from vllm_amd import _lib


def test_strides_of_a_single_row_say_nothing():
    """The C ABI looks at a, out and their row strides only where there is a second row.  (K past what is built is refused behind the strides, and keeps the calls from launching.)"""
    lib, p = _lib.load(), 1 << 20
    k = 131072 + 16
    base = dict(a=p, lda=k, b=p, ldb=k, sa=p, sar=1, sab=1, sb=p, sbk=1, sbn=1, bias=None, out=p, ldc=128, dtype=_lib.VAQ_BF16, m=1, n=128, k=k, stream=None)
    for fields in ({}, dict(lda=1 << 23), dict(lda=k + 8), dict(lda=0), dict(lda=1 << 40), dict(ldc=1), dict(ldc=130), dict(sar=1 << 40)):
        rc = lib.vaq_fp8_block_scaled_mm(*{**base, **fields}.values())
        assert rc == _lib.VAQ_ERR_UNSUPPORTED and "K = 131088" in lib.vaq_last_error().decode(), (fields, rc, lib.vaq_last_error())
    for fields in (dict(lda=1 << 23), dict(lda=k + 8), dict(lda=0), dict(ldc=1), dict(ldc=130)):
        rc = lib.vaq_fp8_block_scaled_mm(*{**base, **fields, "m": 2}.values())
        assert rc != _lib.VAQ_OK and "K = 131088" not in lib.vaq_last_error().decode(), fields
