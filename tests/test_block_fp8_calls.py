"""Host side of the block-scaled FP8 product's calls: strides that say nothing, choice of the plan.  No launch, made-up addresses."""
from __future__ import annotations

import ctypes

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


def test_plans_for_few_rows_have_at_most_eight_blocks_of_rows():
    """On narrow layers with long K, where plans for few rows are the cheapest longest: up to the last row of eight blocks, and not beyond 512 rows."""
    lib, plan = _lib.load(), (ctypes.c_double * 6)()
    few = {}
    for m in (16, 17, 127, 128, 129, 255, 256, 257, 383, 384, 385, 511, 512, 513, 600, 1024, 1025):
        for k in (2048, 8064, 14336):
            for n in (512, 768, 1024):
                assert lib.vaq_fp8_block_plan(m, n, k, plan) == _lib.VAQ_OK
                mb = int(plan[0])
                assert mb == 0 or -(-m // (16 * mb)) <= 8, (m, n, k, list(plan))
                few[m] = few.get(m, 0) + (mb > 0)
    assert all(few[m] for m in few if m <= 512) and not any(few[m] for m in few if m > 512), few


def test_plans_that_the_prices_choose_over_all_recorded_problems():
    """The mean is 1.0106 of the fastest plan's time; without any one of the tile shapes it would be 1.012 .. 1.033."""
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "profiles" / "plan_prices" / "fp8_block.py"
    spec = importlib.util.spec_from_file_location("fp8_block_prices_of_all", path)
    f = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(f)
    by_problem, fitted = f.load()[1], f.load(f.HERE / "fp8_block_fit.csv.gz")[1]
    assert len(by_problem) == 1730 and len(fitted) == 4031 and len(set(by_problem) & set(fitted)) == 3
    assert f.choice(by_problem, *f.tables()).mean() < 1.0115
