"""How combine_tokens_grad rounds: weights times dout in f32, then to ys's type."""
import pytest
import torch

from test_gpu_adapters import cl, gen  # noqa: F401
from test_gpu_adapters_bits import bits

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("y_type,d_type", [(BF16, BF16), (F32, F32), (F32, BF16), (BF16, F32)])
def test_rows_round_to_f32_then_to_their_type(cl, y_type, d_type):
    T, k, cols = 40, 3, 5000
    g = gen(41)
    rows = torch.randperm(T * k, generator=g).int().view(T, k)
    w = torch.rand((T, k), generator=g) * 2 - 1
    w[0, 0], w[1, 1], w[2, 2] = 0.0, -0.0, 1e-38
    dout = torch.randn((T, cols), generator=g).to(d_type)
    dout[:, 0], dout[:, 1], dout[:, 2] = 0.0, -0.0, 1e38
    ys = torch.randn((T * k, cols), generator=g).to(y_type)
    dys, dw = torch.empty_like(ys, device="cuda"), torch.empty((T, k), device="cuda")
    cl.combine_tokens_grad(dout.cuda(), ys.cuda(), rows.cuda(), w.cuda(), dys, dw, top_k=k)
    want = torch.empty_like(ys)
    want[rows.view(-1).long()] = (w[:, :, None] * dout.float()[:, None]).to(y_type).view(T * k, cols)
    assert torch.equal(bits(dys), bits(want))
