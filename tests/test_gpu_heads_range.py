"""The operators on heads at the ends of their numbers' range: rows without an epsilon, rows
far from one, values near the largest."""
import pytest
import torch

import heads_oracle as H
import rmsnorm_tp_b200 as rtp

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def _operands(seed, tokens, hq, hk, d, dtype, odd):
    """q, k and their outputs' gradients: tensors of their own, or at addresses that no
    vector load takes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for heads in (hq, hk, hq, hk):
        x = torch.randn(tokens, heads, d + int(odd), generator=g, device="cuda").to(dtype)
        out.append(x[..., int(odd):])
    w = [(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype) for _ in range(2)]
    rope = rtp.rope_table(4096, d, device="cuda")
    return out, w, rope, torch.randint(4096, (tokens,), generator=g, device="cuda")


def _check_backward(operands, weights, rope, pos, eps, interleaved=False):
    q, k, dq, dk = operands
    got = rtp.qk_norm_rope_backward(dq, dk, q, k, *weights, rope, pos, eps, interleaved)
    for i, (g, x, w) in enumerate(zip((dq, dk), (q, k), weights)):
        dx, s, dw, sw = H.backward(g, x, w, rope, pos, eps, interleaved)
        assert dx.isfinite().all() and dw.isfinite().all()
        H.within(got[i], dx, s, f"dx {i}")
        H.within(got[2 + i], dw, sw, f"dw {i}")


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,hq,hk,d", [(5, 3, 1, 128), (1, 1, 1, 64), (2051, 5, 1, 64), (9, 7, 5, 256)])
def test_backward_without_epsilon(tokens, hq, hk, d, dtype, odd):
    """eps = 0 where the rows leave a part of a warp idle: the idle part adds nothing to dw."""
    _check_backward(*_operands(61, tokens, hq, hk, d, dtype, odd), eps=0.0)


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens", [8, 3000])
@pytest.mark.parametrize("power,eps", [(50, 1e-6), (60, 0.0), (-50, 0.0), (-60, 0.0)])
def test_backward_of_rows_far_from_one(power, eps, tokens, dtype, odd):
    """Rows whose inverse root cubed is no normal fp32 number, while the root and dx are."""
    operands, *rest = _operands(62, tokens, 8, 4, 128, dtype, odd)
    for x in operands[:2]:
        x *= 2.0 ** power
    _check_backward(operands, *rest, eps=eps)
