"""The 8-bit layer's sums on the GPU: slots' rows stay in 32 bits between the down
product and their weighted sum, and layers whose output is f32 add no product in
fewer bits.  Against the 64-bit reference (fp8_ref) with its bound less what such
roundings would add."""
import numpy as np
import pytest
import torch

import fp8_ref as ref
from test_gpu_fp8 import cl, gen, moe_case, moe_ref, run_moe  # noqa: F401 (cl: a fixture)

pytestmark = pytest.mark.gpu


def check(cl, monkeypatch, case, out_dtype, exact, threshold=0.0, tiled=True):
    """The layer within fp8_ref.moe's bound without the slots' bf16 rounding and,
    where exact, without 8-bit sums; an output in bf16 rounds once, by half a step."""
    res = case[-1].to(out_dtype)
    got = run_moe(cl, case, out_dtype, threshold, res, tiled=tiled).double().cpu().numpy()
    with monkeypatch.context() as m:
        m.setattr(ref, "BF16", 0.0)
        if exact:
            m.setattr(ref, "eight_bit_sums", lambda x, w: 0.0)
        want, bound = moe_ref(case, threshold, res)
    if out_dtype == torch.bfloat16:
        bound = bound + ref.BF16 * (np.abs(want) + bound)
    off = np.abs(got - want) - bound
    assert np.all(off <= 0), (off.max(), np.unravel_index(np.argmax(off), off.shape))


# a residual far below the slots, so that the output's own rounding hides nothing
def small_residual(case):
    return (*case[:-1], case[-1] * 2.0 ** -20)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,I,E,k", [(256, 64, 8, 2), (144, 48, 16, 8), (1040, 16, 20, 16),
                                     (64, 80, 3, 1)])
def test_one_token(cl, monkeypatch, H, I, E, k, out_dtype):
    case = small_residual(moe_case(H + I, 1, H, I, E, k, torch.bfloat16))
    check(cl, monkeypatch, case, out_dtype, exact=True)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,I,E,k", [(2, 144, 64, 8, 2), (9, 272, 48, 16, 3), (24, 128, 16, 40, 8),
                                       (60, 64, 32, 96, 4), (100, 32, 16, 700, 8)])
def test_few_rows_per_expert(cl, monkeypatch, T, H, I, E, k, out_dtype):
    """Chunks of 16 rows, of few tokens and of many: exact sums for either output."""
    case = small_residual(moe_case(T + H, T, H, I, E, k, torch.bfloat16))
    check(cl, monkeypatch, case, out_dtype, exact=True)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,I,E,k", [(16, 144, 48, 2, 2), (150, 272, 16, 3, 2),
                                       (300, 64, 144, 5, 4), (140, 32, 32, 1, 1)])
def test_many_rows_per_expert(cl, monkeypatch, T, H, I, E, k, out_dtype):
    """Tiles: 8-bit sums only where the output is bf16, slots in 32 bits always."""
    ids = torch.randint(0, E, (T, k), generator=gen(T), dtype=torch.int32)
    case = small_residual(moe_case(T + H, T, H, I, E, k, torch.bfloat16, ids))
    for tiled in (True, False):
        check(cl, monkeypatch, case, out_dtype, exact=out_dtype == torch.float32, tiled=tiled)
