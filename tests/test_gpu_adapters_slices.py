"""adapters_forward over long rows, K in several slices and one to four tiles of 16 rows a
chunk: outputs whose bounds do not grow with K (adapters_sharp)."""
import pytest
import torch

import adapters_sharp as sharp
from test_gpu_adapters import cl, plan  # noqa: F401

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def forward(cl, case, y_type, base_type):
    a, b, ids, x, base = case
    off, slots = plan(cl, ids, a.shape[0])
    ys = torch.full(base.shape, 77.0, dtype=y_type, device="cuda")
    base = None if base_type is None else base.to(base_type).cuda()
    A = cl.Adapters(a.cuda(), b.cuda())
    return cl.adapters_forward(A, x.cuda(), off, slots, ys, base=base).cpu()


@pytest.mark.parametrize("T,E,R,K,N", sharp.SHAPES)
@pytest.mark.parametrize("x_type", [BF16, F32])
def test_whole_numbers_are_exact(cl, T, E, R, K, N, x_type):
    case = sharp.whole(T, E, R, K, N, x_type)
    for y_type, base_type in ((F32, F32), (BF16, BF16), (F32, BF16)):
        assert sharp.whole_ok(forward(cl, case, y_type, base_type), case), (y_type, base_type)


@pytest.mark.parametrize("T,E,R,K,N", sharp.SHAPES)
def test_picked_columns_come_out_whole(cl, T, E, R, K, N):
    case = sharp.picks(T, E, R, K, N)
    for y_type in (F32, BF16):
        assert sharp.picks_ok(forward(cl, case, y_type, None), case), y_type


@pytest.mark.parametrize("T,E,R,K,N", sharp.SHAPES)
@pytest.mark.parametrize("x_type", [BF16, F32])
def test_random_values(cl, T, E, R, K, N, x_type):
    case = sharp.normal(T, E, R, K, N, x_type)
    for y_type in (F32, BF16):
        assert sharp.normal_ok(forward(cl, case, y_type, None), case), y_type
