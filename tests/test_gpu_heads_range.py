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


@pytest.mark.parametrize("batch,n", [(1, 300), (300, 600), (3, 3000)])
@pytest.mark.parametrize("dtype,held,group,d", [(BF16, BF16, 8, 128), (BF16, E4M3, 8, 128), (BF16, BF16, 16, 64), (BF16, E4M3, 12, 256),
                                                (F32, F32, 2, 64), (F32, E4M3, 2, 64)])
def test_attention_of_values_near_the_largest(batch, n, dtype, held, group, d):
    """The first token and a late one have values near the largest of bf16 and fp32, and the
    late one's score passes the others' by a little less than the softmax's reference follows
    at once: the output is finite, and so is each of its sums."""
    page, at = 64, n - 20
    k, v = (torch.zeros(-(-n // page), 1, page, d, device="cuda") for _ in range(2))
    k[at // page, 0, at % page, 0] = 5.5                         # 5.5 log2(e) = 7.93
    row = torch.where(torch.arange(d, device="cuda") % 2 == 0, 1.5, -1.25) * 2.0 ** 126
    v[at // page, 0, at % page] = v[0, 0, 0] = row
    if held == E4M3:
        one, vs = torch.ones(k.shape[:3], device="cuda"), torch.ones(v.shape[:3], device="cuda")
        vs[at // page, 0, at % page] = vs[0, 0, 0] = 2.0 ** 119
        cache = rtp.PagedKVCache.from_tensors(k.to(E4M3), (v / vs[..., None]).to(E4M3), one, vs)
    else:
        cache = rtp.PagedKVCache.from_tensors(k.to(held), v.to(held))
    q = torch.zeros(batch, group, d, dtype=dtype, device="cuda")
    q[..., 0] = 1
    table = torch.arange(k.shape[0], dtype=torch.int32, device="cuda").expand(batch, -1)
    got, lse = rtp.paged_attention(q, cache, table, torch.full((batch,), n, dtype=torch.int32, device="cuda"), 1.0,
                                   return_lse=True)
    p = torch.exp(torch.tensor([5.5], dtype=torch.float64, device="cuda"))
    want = ((p + 1) / (p + n - 1) * row.double()).expand(batch, group, d)
    # the weights: sums and exponentials of fp32, 2^-11 where the numerators are one fp16 part
    # (the two parts of bf16: 2^-16)
    rel = (2 * n + 128) * H.U32 + (2.0 ** -11 if held == E4M3 and dtype == BF16 else 2.0 ** -16 if held == BF16 else 0.0)
    H.within(got, want, rel * want.abs(), "out")
    assert (lse.double() - torch.log(p + n - 1)).abs().max() <= (n + 128) * H.U32


def test_attention_of_an_infinite_value_without_weight():
    """An infinity in V whose token's weight no 16-bit part holds does not vanish."""
    k, v = torch.zeros(1, 1, 64, 64, device="cuda", dtype=F16), torch.ones(1, 1, 64, 64, device="cuda", dtype=F16)
    k[0, 0, 0, 0], v[0, 0, 1, 3] = 35.0, float("inf")            # e^-35 of the heaviest: under 2^-50
    q = torch.zeros(1, 8, 64, dtype=F16, device="cuda")
    q[..., 0] = 1
    got = rtp.paged_attention(q, rtp.PagedKVCache.from_tensors(k, v), torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                              torch.full((1,), 64, dtype=torch.int32, device="cuda"), 1.0)
    assert not got[..., 3].isfinite().any() and (got[..., :3] == 1).all() and (got[..., 4:] == 1).all()
