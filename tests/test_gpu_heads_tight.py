"""The attention against the formula in 64 bits within the precision that its kernels hold
the softmax's weights to, for every shape of kernel; the backward in the projection's layouts."""
import itertools
import random

import pytest
import torch

import heads_oracle as H
import rmsnorm_tp_b200 as rtp
from test_gpu_heads import SHAPES, _filled, _gen, _heads, _normal, _positions, _table, _weights

pytestmark = pytest.mark.gpu

EPS = 1e-6
BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def _weight_step(dtype, held, d):
    """(relative, absolute) error of a weight on its way to the products, the second as a part
    of the heaviest one: two bf16 parts 2^-16; two fp16 parts 2^-20, one (e4m3 beside bf16)
    2^-11, the smallest of them half of fp16's smallest number, 2^-25, where the heaviest is at
    least 2^7. fp32, and head_dims of the plain kernel: none."""
    if dtype == F32 or d not in (64, 96, 128, 192, 256):
        return 0.0, 0.0
    if held == BF16:
        return 2.0 ** -16, 0.0
    return 2.0 ** -11 if held == E4M3 and dtype == BF16 else 2.0 ** -20, 2.0 ** -32


def _attend(q, cache, table, lens, scale):
    """heads_oracle's attention, its bound with the weights' errors above."""
    d, held = q.shape[-1], cache.dtype
    out, fp32, lse, lslop = H.attend(q, cache, table, lens, scale, 0.0)
    around = (H.attend(q, cache, table, lens, scale, 2.0 ** -20)[1] - fp32) * 2.0 ** 20   # sum p |v| / l
    rel, part = _weight_step(q.dtype, held, d)
    slop = fp32 + rel * around
    for b in range(q.shape[0] if part else 0):
        n = min(max(int(lens[b]), 0), table.shape[1] * cache.page_size)
        t = torch.arange(n, device=q.device)
        pages = table[b].long()[t // cache.page_size]
        live = (pages >= 0) & (pages < cache.num_pages)
        pages, off = pages[live], (t % cache.page_size)[live]
        if not pages.numel():
            continue
        k = H.rows_of(cache, "k", pages, off).transpose(0, 1).repeat_interleave(q.shape[1] // cache.num_kv_heads, 0)
        p = torch.softmax(torch.einsum("hd,hnd->hn", q[b].double(), k) * scale, -1)
        # each weight (e4m3: times its row's scale) off by `part` of the heaviest, times an element (a code)
        if held == E4M3:
            vs = cache.v_scale[pages, :, off].double().t().repeat_interleave(q.shape[1] // cache.num_kv_heads, 0)
            codes = cache.v.view(torch.uint8)[pages, :, off].view(E4M3).double().abs().amax()
            most = (p * vs).amax(-1) * codes
        else:
            most = p.amax(-1) * cache.v[pages, :, off].double().abs().amax()
        slop[b] += (pages.numel() * part * most)[:, None]
    return out, slop, lse, lslop


def _check(q, cache, table, lens, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    got, lse = rtp.paged_attention(q, cache, table, lens, scale, return_lse=True)
    out, slop, want, lslop = _attend(q, cache, table, lens, scale)
    # past the type's largest by half a step a value rounds to infinity
    most = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    over = torch.isinf(got) & (out.abs() + slop >= most) & (got.sign() == out.sign())
    H.within(got.masked_fill(over, 0), out.masked_fill(over, 0), slop.masked_fill(over, 0), "out")
    live = ~torch.isneginf(want)
    assert torch.equal(torch.isneginf(lse), ~live)
    H.within(lse[live], want[live], lslop[live], "lse")


TYPES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3)]


@pytest.mark.parametrize("width", [None, 400])
@pytest.mark.parametrize("dtype,held", TYPES)
@pytest.mark.parametrize("d,group,page", list(itertools.chain(
    ((d, g, 16) for d in (64, 96, 128, 192, 256) for g in (1, 8, 9, 16)),
    ((d, g, p) for d in (96, 192) for g, p in ((12, 7), (16, 64), (33, 32))))))
def test_every_kernel_within_its_precision(d, group, page, dtype, held, width):
    lens = [0, 1, 33, 64, 129, 500, 15]
    pages = sum(-(-n // page) for n in lens) + 3
    cache = _filled(71, pages, page, 2, d, held)
    q = (2 * _normal(_gen(72), len(lens), 2 * group, d)).to(dtype)
    _check(q, cache, _table(71, lens, page, pages, width=width and max(width, -(-500 // page))),
           torch.tensor(lens, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype,held", [(F16, F16), (F16, E4M3), (BF16, BF16)])
@pytest.mark.parametrize("group", [8, 16])
def test_a_weights_second_part(group, dtype, held):
    """Values of +-1 whose weighted sums nearly cancel: what is left shows the weights to the
    last bits that the kernels hold, where one 16-bit part of each would be seen to be one."""
    n, d, page = 12, 64, 16
    s = -torch.arange(n, dtype=torch.float64) / 13 + 1e-3
    s = s.to(held if held != E4M3 else F32).double()
    p = torch.exp(s - s.max())
    signs = torch.tensor(list(itertools.product((1.0, -1.0), repeat=n)), dtype=torch.float64)
    sums = (signs * p).sum(1) / p.sum()
    best = sums.abs().argsort()[:d]
    want = sums[best].cuda()
    k, v = torch.zeros(1, 1, page, d, device="cuda"), torch.zeros(1, 1, page, d, device="cuda")
    v[0, 0, :n] = signs[best].t().float().cuda()
    scales = ()
    if held == E4M3:
        k[0, 0, :n, 0] = 1
        scales = torch.ones(1, 1, page, device="cuda"), torch.ones(1, 1, page, device="cuda")
        scales[0][0, 0, :n] = s.float().cuda()
    else:
        k[0, 0, :n, 0] = s.float().cuda()
    cache = rtp.PagedKVCache.from_tensors(k.to(held), v.to(held), *scales)
    q = torch.zeros(1, group, d, dtype=dtype, device="cuda")
    q[..., 0] = 1
    got = rtp.paged_attention(q, cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                              torch.tensor([n], dtype=torch.int32, device="cuda"), 1.0)
    # a score is one exact product; its scaling, the exponential and the sums as in heads_oracle
    rel = (2 * 16 + 2 * n + 64) * H.U32 + _weight_step(dtype, held, d)[0] + n * 2.0 ** -32
    H.within(got, want.expand(1, group, d), torch.full((1, group, d), rel, dtype=torch.float64, device="cuda"), "out")
    # the case can tell: weights of one part (of the type of the products) leave the bound
    one = (signs[best] * p.to(F16 if held != BF16 else BF16).double()).sum(1) / p.sum()
    bound = H.half_step(dtype) * sums[best].abs() + 2 * rel
    assert ((one - sums[best]).abs() > bound).sum() > d // 4


@pytest.mark.parametrize("seed", range(80))
def test_random_calls(seed):
    """Sizes, types and lengths over the whole range, scores and values up to some decades apart."""
    rng = random.Random(seed)
    dtype, held = rng.choice(TYPES + [(F32, F32), (F32, E4M3)])
    hk, group, d = rng.randint(1, 4), rng.choice([1, 2, 3, 5, 7, 8, 9, 12, 16, 17, 24]), 16 * rng.randint(1, 16)
    if rng.random() < 0.6:
        d = rng.choice([64, 96, 128, 192, 256])
    page, batch = rng.choice([1, 7, 16, 32, 48, 64, 128]), rng.choice([1, 2, 5, 30])
    most = rng.choice([3, 70, 600, 4000 // batch])
    lens = [rng.randint(0, most) for _ in range(batch)]
    pages = sum(-(-n // page) for n in lens) + 2
    cache = _filled(100 + seed, pages, page, hk, d, held)
    far = rng.choice([0.0, 1.0, 2.5])
    spread = torch.exp(far * _normal(_gen(seed), pages, hk, page))
    if held == E4M3:
        cache.v_scale *= spread
    else:
        cache.v.mul_(spread[..., None].clamp(1e-3, 1e3).to(held))
    q = (rng.choice([0.3, 2.0, 8.0]) * _normal(_gen(200 + seed), batch, hk * group, d)).to(dtype)
    table = _table(300 + seed, lens, page, pages, width=rng.choice([None, -(-most // page) + 600 // page + 1]))
    _check(q, cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), rng.choice([None, 1.0 / d, -0.1]))


@pytest.mark.parametrize("layout", ["blocks", "heads_first"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES + [(4099, 8, 2, 64, 64), (700, 32, 8, 128, 128)], ids=str)
def test_backward_in_the_projections_layouts(shape, dtype, layout):
    tokens, hq, hk, d, r = shape
    q, k, _ = _heads(5, tokens, hq, hk, d, dtype, layout)
    dq, dk, _ = _heads(6, tokens, hq, hk, d, dtype, layout)
    weights = _weights(5, d, dtype)
    rope, pos = rtp.rope_table(4096, r, device="cuda"), _positions(5, tokens, 4096)
    for interleaved in (False, True):
        got = rtp.qk_norm_rope_backward(dq, dk, q, k, *weights, rope, pos, EPS, interleaved)
        for i, (g, x, w) in enumerate(zip((dq, dk), (q, k), weights)):
            dx, s, dw, sw = H.backward(g, x, w, rope, pos, EPS, interleaved)
            H.within(got[i], dx, s, f"dx {i} {interleaved}")
            H.within(got[2 + i], dw, sw, f"dw {i} {interleaved}")
