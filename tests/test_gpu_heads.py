"""GPU parity of the operators on query / key heads, the paged cache and the single-token
attention against the formulas in 64 bits (heads_oracle), at sizes, strides, masks and
values where they can go wrong; the run of them together between the package's norms."""
import math
import subprocess
import sys

import pytest
import torch

import heads_oracle as H
import rmsnorm_tp_b200 as rtp
from conftest import ROOT

pytestmark = pytest.mark.gpu

EPS = 1e-6
BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *n):
    return torch.randn(*n, generator=g, device="cuda")


def _heads(seed, tokens, hq, hk, d, dtype, layout="blocks"):
    """q, k, v as column blocks of one matrix, as tensors of their own, with heads before
    tokens, or at addresses that no vector load takes."""
    g = _gen(seed)
    x = _normal(g, tokens, (hq + 2 * hk) * d) * torch.where(torch.rand((hq + 2 * hk) * d, generator=g, device="cuda")
                                                            < 0.02, 30.0, 1.0)
    x = x.to(dtype)
    if layout == "odd":
        x = torch.cat([x.new_zeros(tokens, 1), x, x.new_zeros(tokens, 2)], 1)[:, 1:-2]
    q, k, v = (t.unflatten(1, (-1, d)) for t in x.split([hq * d, hk * d, hk * d], 1))
    if layout == "own":
        q, k, v = (t.contiguous() for t in (q, k, v))
    if layout == "heads_first":
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    return q, k, v


def _weights(seed, d, dtype):
    g = _gen(seed + 50)
    return [(1 + 0.2 * _normal(g, d)).to(dtype) for _ in range(2)]


def _positions(seed, tokens, most):
    return torch.randint(most, (tokens,), generator=_gen(seed + 60), device="cuda")


SHAPES = [   # tokens, q heads, kv heads, head_dim, rotary_dim
    (1, 1, 1, 64, 64), (1, 32, 8, 128, 128), (5, 8, 1, 128, 128), (333, 7, 3, 96, 48), (64, 8, 2, 256, 256),
    (17, 6, 2, 192, 64), (130, 12, 4, 80, 32), (9, 4, 4, 32, 32), (33, 3, 1, 50, 24), (3, 2, 2, 2, 2),
    (7, 5, 5, 512, 512), (1025, 16, 2, 128, 64), (40, 2, 1, 33, 6)]


@pytest.mark.parametrize("layout", ["blocks", "heads_first", "odd"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm_and_rotation(shape, dtype, layout):
    tokens, hq, hk, d, r = shape
    q, k, _ = _heads(1, tokens, hq, hk, d, dtype, layout)
    qw, kw = _weights(1, d, dtype)
    rope, pos = rtp.rope_table(4096, r, device="cuda"), _positions(1, tokens, 4096)
    for interleaved in (False, True):
        for weights in ((qw, kw), (None, None)):
            got = rtp.qk_norm_rope(q, k, *weights, rope, pos, EPS, interleaved)
            for x, w, y, name in zip((q, k), weights, got, "qk"):
                H.within(y, *H.forward(x, w, rope, pos, EPS, interleaved), f"{name} {interleaved} {w is None}")


def test_in_place_in_the_projection_and_into_views():
    q, k, v = _heads(2, 77, 8, 2, 128, BF16)
    base = q._base if q._base is not None else q
    qw, kw = _weights(2, 128, BF16)
    rope, pos = rtp.rope_table(512, 128, device="cuda"), _positions(2, 77, 512)
    want = rtp.qk_norm_rope(q, k, qw, kw, rope, pos, EPS)
    v0 = v.clone()
    wide = torch.full((77, 10, 160), 7.0, dtype=BF16, device="cuda")
    rtp.qk_norm_rope(q, k, qw, kw, rope, pos, EPS, q_out=wide[:, :8, 16:144], k_out=wide[:, 8:, 16:144])
    assert torch.equal(wide[:, :8, 16:144], want[0]) and torch.equal(wide[:, 8:, 16:144], want[1])
    assert (wide[:, :, :16] == 7).all() and (wide[:, :, 144:] == 7).all()
    got = rtp.qk_norm_rope(q, k, qw, kw, rope, pos, EPS, q_out=q, k_out=k)
    assert got[0].data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(v, v0) and base.numel() >= q.numel()
    # an offset that keeps no vector aligned: the same values, in place
    q, k, _ = _heads(2, 77, 3, 2, 50, F16, "odd")
    qw, kw = _weights(2, 50, F16)
    rope = rtp.rope_table(512, 20, device="cuda")
    want = rtp.qk_norm_rope(q, k, qw, kw, rope, pos, EPS, True)
    rtp.qk_norm_rope(q, k, qw, kw, rope, pos, EPS, True, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("d,r", [(128, 128), (96, 48), (50, 20)])
def test_positions_outside_the_table_zero_rows_and_values_that_are_not_numbers(d, r):
    q, k, _ = _heads(3, 6, 4, 2, d, BF16)
    q, k = q.clone(), k.clone()
    q[1] = 0
    q[2, 1, 3] = float("nan")
    k[3, 0, 5] = float("inf")
    rope, pos = rtp.rope_table(10, r, device="cuda"), torch.tensor([0, 9, 3, 4, -1, 10], device="cuda")
    w, _ = _weights(3, d, BF16)
    got = rtp.qk_norm_rope(q, k, w, w, rope, pos, EPS)
    for x, y in zip((q, k), got):
        H.within(y, *(t.nan_to_num() if i else t for i, t in enumerate(H.forward(x, w, rope, pos, EPS, False))), "y")
    assert got[0][4:, :, :r].isnan().all() and not got[0][4:, :, r:].isnan().any()
    assert (got[0][1] == 0).all()


def test_expanded_inputs_and_no_tokens():
    q, k, _ = _heads(4, 1, 4, 4, 64, BF16)
    q, k = q.expand(9, -1, -1), k[:, :1].expand(9, 4, -1)
    w, _ = _weights(4, 64, BF16)
    rope, pos = rtp.rope_table(64, 64, device="cuda"), _positions(4, 9, 64)
    for x, y in zip((q, k), rtp.qk_norm_rope(q, k, w, w, rope, pos, EPS)):
        H.within(y, *H.forward(x, w, rope, pos, EPS, False), "expanded")
    none = rtp.qk_norm_rope(q[:0], k[:0], w, w, rope, pos[:0], EPS)
    assert none[0].shape == (0, 4, 64)
    grads = rtp.qk_norm_rope_backward(q[:0], k[:0], q[:0], k[:0], w, w, rope, pos[:0], EPS)
    torch.cuda.synchronize()
    assert (grads[2] == 0).all() and (grads[3] == 0).all() and grads[0].numel() == 0


@pytest.mark.parametrize("layout", ["own", "odd"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES + [(4099, 8, 2, 64, 64)], ids=str)
def test_backward(shape, dtype, layout):
    tokens, hq, hk, d, r = shape
    q, k, _ = _heads(5, tokens, hq, hk, d, dtype, layout)
    dq, dk, _ = _heads(6, tokens, hq, hk, d, dtype, layout)
    qw, kw = _weights(5, d, dtype)
    rope, pos = rtp.rope_table(4096, r, device="cuda"), _positions(5, tokens, 4096)
    for interleaved in (False, True):
        for weights in ((qw, kw), (None, None)):
            got = rtp.qk_norm_rope_backward(dq, dk, q, k, *weights, rope, pos, EPS, interleaved)
            again = rtp.qk_norm_rope_backward(dq, dk, q, k, *weights, rope, pos, EPS, interleaved)
            for i, (g, x, w) in enumerate(zip((dq, dk), (q, k), weights)):
                dx, s, dw, sw = H.backward(g, x, w, rope, pos, EPS, interleaved)
                H.within(got[i], dx, s, f"dx {i} {interleaved}")
                assert torch.equal(got[i], again[i])
                if w is None:
                    assert got[2 + i] is None
                else:
                    H.within(got[2 + i], dw, sw, f"dw {i} {interleaved}")
                    assert torch.equal(got[2 + i], again[2 + i])


def test_autograd_with_shared_and_broadcast_inputs():
    """Autograd around the kernels, a query expanded over tokens and a weight that both norms
    share: their gradients are the sums of the formula's."""
    tokens, h, d = 21, 4, 64
    rope, pos = rtp.rope_table(64, d, device="cuda"), _positions(7, tokens, 64)
    q, k, _ = _heads(7, tokens, h, 2, d, F32, "own")
    gq, gk, _ = _heads(8, tokens, h, 2, d, F32, "own")
    one = q[:1].clone().requires_grad_()
    k = k.clone().requires_grad_()
    w = _weights(7, d, F32)[0].clone().requires_grad_()
    y = rtp.qk_norm_rope_with_grad(one.expand(tokens, -1, -1), k, w, w, rope, pos, EPS)
    ((y[0] * gq).sum() + (y[1].transpose(0, 1) * gk.transpose(0, 1)).sum()).backward()
    dq, sq, dwq, s1 = H.backward(gq, one.detach().expand(tokens, -1, -1), w.detach(), rope, pos, EPS, False)
    dk, sk, dwk, s2 = H.backward(gk, k.detach(), w.detach(), rope, pos, EPS, False)
    # torch's own sums of `tokens` rows and of the two weights come on top
    H.within(k.grad, dk, sk, "dk")
    H.within(one.grad, dq.sum(0, keepdim=True), sq.sum(0, keepdim=True) + (tokens + 2) * H.U32 * dq.abs().sum(0), "dq")
    H.within(w.grad, dwq + dwk, s1 + s2 + 4 * H.U32 * (dwq.abs() + dwk.abs()), "dw")
    with pytest.raises(RuntimeError):                   # no gradient of the gradient
        z = rtp.qk_norm_rope_with_grad(k, k, w, w, rope, pos, EPS)[0].square().sum()
        torch.autograd.grad(torch.autograd.grad(z, k, create_graph=True)[0].sum(), k)
    # only one output used: the other's gradient is zero
    a, b = (t.detach().clone().requires_grad_() for t in (q, k))
    rtp.qk_norm_rope_with_grad(a, b, None, None, rope, pos, EPS)[0].sum().backward()
    assert (b.grad == 0).all() and a.grad.abs().sum() > 0


# ---- cache ---------------------------------------------------------------------------

def _filled(seed, pages, page, heads, d, dtype):
    """A cache whose every row is in use."""
    g = _gen(seed)
    k, v = _normal(g, pages, heads, page, d), _normal(g, pages, heads, page, d)
    if dtype != E4M3:
        return rtp.PagedKVCache.from_tensors(k.to(dtype), v.to(dtype))
    v = v * torch.exp(2 * _normal(g, pages, heads, page, 1))
    rows = []
    for x in (k, v):
        most = x.abs().amax(-1, keepdim=True)
        rows.append(((x * (448.0 / most)).clamp(-448, 448).to(E4M3), (most / 448.0).squeeze(-1)))
    return rtp.PagedKVCache.from_tensors(rows[0][0], rows[1][0], rows[0][1], rows[1][1])


def _state(cache):
    """The bits of the cache's tensors, an element each."""
    bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}
    return [t.view(bits[t.element_size()]).clone()
            for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]


@pytest.mark.parametrize("dtype,held", [(BF16, E4M3), (F16, E4M3), (F32, E4M3), (BF16, BF16), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("layout", ["blocks", "odd"])
@pytest.mark.parametrize("tokens,hq,hk,d,r,page", [(1, 8, 1, 128, 128, 64), (70, 8, 2, 64, 64, 16), (257, 6, 3, 96, 48, 7),
                                                   (33, 4, 1, 256, 256, 1), (40, 3, 3, 80, 32, 48), (19, 2, 2, 16, 6, 5)])
def test_write_then_read(tokens, hq, hk, d, r, page, layout, dtype, held):
    pages = -(-tokens // page) + 3
    cache = _filled(11, pages, page, hk, d, held)
    before = _state(cache)
    q, k, v = _heads(11, tokens, hq, hk, d, dtype, layout)
    qw, kw = _weights(11, d, dtype)
    rope, pos = rtp.rope_table(2048, r, device="cuda"), _positions(11, tokens, 2048)
    slots = torch.randperm(pages * page, generator=_gen(11), device="cuda")[:tokens].contiguous()
    slots[tokens // 2::5] = -1                                # padding
    slots[tokens // 3::11] = pages * page                     # behind the cache
    inter = page == 7
    q_out = rtp.qk_norm_rope_write(q, k, v, qw, kw, rope, pos, cache, slots, EPS, inter)
    H.within(q_out, *H.forward(q, qw, rope, pos, EPS, inter), "q")
    live = (slots >= 0) & (slots < pages * page)
    at, off = slots[live] // page, slots[live] % page
    want_k, slop = H.forward(k, kw, rope, pos, EPS, inter)
    for name, want, s in (("k", want_k[live], slop[live]), ("v", v.double()[live], torch.zeros_like(slop[live]))):
        rows = getattr(cache, name)
        if held == E4M3 and live.any():
            codes = rows.view(torch.uint8)[at, :, off].view(E4M3)
            H.within_e4m3(codes, getattr(cache, name + "_scale")[at, :, off], want, s, name)
        elif live.any():
            H.within(rows[at, :, off], want, s, name)
    # every other row as it was
    kept = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    kept[at, off] = False
    i, j = kept.nonzero(as_tuple=True)
    for old, new in zip(before, _state(cache)):
        assert torch.equal(old[i, :, j], new[i, :, j])
    # read back: the values the rows stand for, rounded once; zeros outside the cache
    for out in (F32, BF16, F16):
        for name, got in zip("kv", cache.read(slots, out)):
            rows = H.rows_of(cache, name, (slots // page).clamp(0, pages - 1), slots % page)
            H.within(got, torch.where(live[:, None, None], rows, 0.0), 2 * H.U32 * rows.abs(), f"read {name}")


def test_rows_that_scales_cannot_hold():
    """Zeros, numbers near the smallest, infinities and NaN through an e4m3 cache."""
    d, cache = 64, rtp.PagedKVCache(2, 8, 1, 64, E4M3)
    v = torch.ones(6, 1, d, device="cuda")
    v[0] = 0
    v[1] = 2.0 ** -120
    v[2, 0, 1] = float("inf")
    v[3, 0, 2] = float("nan")
    v[4] = 3e38
    v[5, 0, 0] = -448.0
    rope, pos = rtp.rope_table(8, d, device="cuda"), torch.zeros(6, dtype=torch.int64, device="cuda")
    slots = torch.arange(6, device="cuda") + 5
    for layout in ("own", "odd"):
        x = v if layout == "own" else torch.cat([v.new_zeros(6, 1, 1), v], 2)[:, :, 1:]
        rtp.qk_norm_rope_write(v, v, x, None, None, rope, pos, cache, slots, EPS)
        got = cache.read(slots, F32)[1][:, 0]
        assert (got[0] == 0).all() and (got[1].abs() <= 2.0 ** -100).all()
        assert got[2].isnan().all()                      # the scale of an infinite row is infinite
        assert got[3, 2].isnan() and (got[3, :2] == 1).all()
        assert (got[4] / 3e38 - 1).abs().max() <= 2.0 ** -20
        assert got[5, 0] == -448 and (got[5, 1:] == 1).all()
    torch.cuda.synchronize()


def test_read_of_no_slots_and_fresh_cache():
    cache = rtp.PagedKVCache(3, 16, 2, 64, E4M3)
    k, v = cache.read(torch.arange(-2, 50, device="cuda"))
    assert k.dtype == BF16 and (k == 0).all() and (v == 0).all()
    assert cache.read(torch.empty(0, dtype=torch.int64, device="cuda"))[0].shape == (0, 2, 64)


# ---- attention -------------------------------------------------------------------------

def _p_step(dtype, held):
    """Half step of the type the softmax's numerators are held in before the product with V:
    fp16 for fp16 and e4m3 caches, two bf16 parts (together 2^-16) for bf16."""
    return 2.0 ** -16 if held == BF16 else 0.0 if held == F32 or dtype == F32 else 2.0 ** -11


def _table(seed, lens, page, pages, width=None):
    used = [-(-n // page) for n in lens]
    order = torch.randperm(pages, generator=_gen(seed), device="cuda").to(torch.int32)
    table = torch.full((len(lens), width or max(1, max(used))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return table


def _check_attention(q, cache, table, lens, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    got, lse = rtp.paged_attention(q, cache, table, lens, scale, return_lse=True)
    out, slop, want, lslop = H.attend(q, cache, table, lens, scale, _p_step(q.dtype, cache.dtype))
    H.within(got, out, slop, "out")
    assert torch.equal(torch.isneginf(lse), torch.isneginf(want))
    live = ~torch.isneginf(want)
    H.within(lse[live], want[live], lslop[live], "lse")
    return got, lse


TYPES = [(BF16, BF16), (F16, F16), (F32, F32), (BF16, E4M3), (F16, E4M3), (F32, E4M3)]


@pytest.mark.parametrize("dtype,held", TYPES)
@pytest.mark.parametrize("hk,group,d,page", [(1, 8, 128, 64), (2, 1, 64, 16), (3, 5, 96, 7), (1, 16, 256, 32),
                                             (2, 4, 192, 48), (1, 20, 128, 1), (2, 7, 80, 16), (1, 40, 64, 128),
                                             (1, 3, 16, 3)])
def test_attention(dtype, held, hk, group, d, page):
    lens = [0, 1, 2, 63, 64, 65, 300, 17, 1000]
    pages = sum(-(-n // page) for n in lens) + 3
    cache = _filled(21, pages, page, hk, d, held)
    q = (2 * _normal(_gen(22), len(lens), hk * group, d)).to(dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got, lse = _check_attention(q, cache, _table(21, lens, page, pages), lens_t)
    assert (got[0] == 0).all() and torch.isneginf(lse[0]).all()


@pytest.mark.parametrize("dtype,held", [(BF16, BF16), (F16, E4M3), (F32, F32)])
@pytest.mark.parametrize("lens", [[5000], [1], [0], [9000, 1, 0, 64], [129] * 300, [37 * i % 700 for i in range(70)]],
                         ids=lambda l: f"{len(l)}x{max(l)}")
def test_attention_divided_over_the_length(dtype, held, lens):
    page, hk, d = 16, 1, 128
    pages = sum(-(-n // page) for n in lens) + 1
    cache = _filled(23, pages, page, hk, d, held)
    q = (2 * _normal(_gen(24), len(lens), 8, d)).to(dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    a = _check_attention(q, cache, _table(23, lens, page, pages), lens_t)
    b = rtp.paged_attention(q, cache, _table(23, lens, page, pages), lens_t, return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])           # no order that changes
    # a wider table than any sequence needs changes only how the work is divided
    c, _ = _check_attention(q, cache, _table(23, lens, page, pages, width=700), lens_t)


@pytest.mark.parametrize("dtype,held", [(BF16, BF16), (F16, F16), (BF16, E4M3), (F32, F32)])
def test_attention_masked_places(dtype, held):
    """Bad pages and values that are not numbers where no token lies; lengths out of range;
    strided queries and tables."""
    page, hk, d, lens = 16, 2, 128, [40, 33, 64, 50, 64]
    cache = _filled(25, 30, page, hk, d, held)
    table = _table(25, lens, page, 29, width=4)
    junk = torch.full((), float("nan"), device="cuda")
    for t in ((cache.k_scale, cache.v_scale) if held == E4M3 else (cache.k, cache.v)):
        t[table[0, 2].long(), :, 8:] = junk                     # behind the last token of its page
        t[29] = float("inf")                                   # a page that no sequence has
    if held == E4M3:
        cache.k.view(torch.uint8)[table[1, 2].long(), :, 1:] = 0x7F      # codes that are NaN
        cache.v.view(torch.uint8)[table[1, 2].long(), :, 1:] = 0xFF
    table[3, 1] = -1
    table[2, 0] = 30                                           # outside the cache: left out
    table[4] = -5                                              # a row with nothing left
    lens_t = torch.tensor([40, 33, 64, 50, 64], dtype=torch.int32, device="cuda")
    wide = _normal(_gen(26), 5, 3, 8, d).to(dtype)
    got, lse = _check_attention(wide[:, 1, ::2], cache, table, lens_t)
    assert (got[4] == 0).all() and torch.isneginf(lse[4]).all()
    wide_table = torch.full((5, 9), 7, dtype=torch.int32, device="cuda")
    wide_table[:, 2:6] = table
    again = rtp.paged_attention(wide[:, 1, ::2], cache, wide_table[:, 2:6], lens_t)
    assert torch.equal(again, got)
    out_of_range = torch.tensor([-3, 1 << 30, 64, -(1 << 31), 64], dtype=torch.int32, device="cuda")
    table[1, 3] = table[1, 2]
    cut = out_of_range.clamp(0, 64)
    if held != E4M3:      # sequence 1 now reads whole pages: keep numbers in them
        _check_attention(wide[:, 1, ::2], cache, table, cut)
    a = rtp.paged_attention(wide[:, 1, ::2], cache, table, out_of_range)
    b = rtp.paged_attention(wide[:, 1, ::2], cache, table, cut)
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    none = rtp.paged_attention(wide[:, 1, ::2], cache, table[:, :0], lens_t, return_lse=True)
    assert (none[0] == 0).all() and torch.isneginf(none[1]).all()
    assert rtp.paged_attention(wide[:0, 1], cache, table[:0], lens_t[:0]).shape == (0, 8, d)


@pytest.mark.parametrize("dtype,held", TYPES)
def test_attention_large_and_small_numbers(dtype, held):
    """Scores far apart (one token takes all), far from zero, equal, infinite; values whose
    scales are far apart, the attended token's the smallest; -inf and NaN keys."""
    page, d, n = 16, 64, 200
    cache = _filled(27, 20, page, 1, d, held)
    table, lens = _table(27, [n], page, 20), torch.tensor([n], dtype=torch.int32, device="cuda")
    q = _normal(_gen(28), 1, 4, d).to(dtype)
    for scale in (0.0, 40.0, -3.0, 1e-6):
        _check_attention(q, cache, table, lens, scale)
    if held == E4M3:
        cache.v_scale *= 2.0 ** 12
        row = table[0, 6].long()
        cache.v_scale[row, :, 4] *= 2.0 ** -20                 # the token that takes nearly all the weight
        cache.k.view(torch.uint8)[row, :, 4] = (q[:, :1].float() / q[:, :1].float().abs().max() * 448).to(E4M3).view(torch.uint8)[0]
        cache.k_scale[row, :, 4] = 1.0
        _check_attention(q, cache, table, lens, 1.0)
        cache.v_scale *= 2.0 ** -60
        _check_attention(q, cache, table, lens, 0.2)
    else:
        big = cache.k.abs().max().item()
        cache.k[table[0, 3].long(), :, 2] = -float("inf")
        cache.v[table[0, 5].long(), :, 2, 3] = float("inf")
        got = rtp.paged_attention(q.abs() + 0.1, cache, table, lens)
        assert torch.isinf(got[..., 3]).all() and not torch.isnan(got).any() and big > 0
        cache.k[table[0, 1].long(), :, 3, 5] = float("nan")
        got, lse = rtp.paged_attention(q, cache, table, lens, return_lse=True)
        assert got.isnan().all() and lse.isnan().all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_elements_that_the_heaviest_token_lacks(dtype):
    """Half of the heaviest token's elements are 0, and its V scale is 64 times the others':
    these elements are made of tokens whose weights lie near fp16's smallest number."""
    d, page = 128, 16
    cache = _filled(51, 2, page, 1, d, E4M3)
    n, want_s = 3, torch.tensor([16.0, 8.0, 7.0], device="cuda")
    cache.k[0, 0, :n] = torch.ones(n, d, device="cuda").to(E4M3)
    cache.k_scale[0, 0, :n] = want_s / d
    codes = 448 * torch.rand(n, d, generator=_gen(52), device="cuda")
    codes[0, ::2] = 0
    cache.v[0, 0, :n] = codes.to(E4M3)
    cache.v_scale[0, 0, :n] = torch.tensor([0.5, 1 / 128, 1 / 128], device="cuda")
    q = torch.ones(1, 8, d, device="cuda", dtype=dtype)
    got = rtp.paged_attention(q, cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                              torch.tensor([n], dtype=torch.int32, device="cuda"), 1.0)
    p, vs = torch.softmax(want_s.double(), 0), cache.v_scale[0, 0, :n].double()
    v = codes.to(E4M3).double() * vs[:, None]
    want = (p[:, None] * v).sum(0).expand(1, 8, d)
    # the scores are off by (d + 8) units of 2^-24 at most; a weight by half a step of its
    # type, or, where it is small, by 2^-25 beside a heaviest one of 2^7 (codes up to 448)
    rel = 2 * (d + 24) * H.U32 * 16 + 64 * H.U32 + (2.0 ** -11 if dtype == BF16 else 2.0 ** -16)
    slop = (rel * (p[:, None] * v.abs()).sum(0) + (n - 1) * 2.0 ** -32 * 448 * (p * vs).max()).expand(1, 8, d)
    H.within(got, want, slop, "out")


@pytest.mark.parametrize("held", [F16, E4M3])
def test_attention_many_tokens_without_weight(held):
    """One token takes all the weight and its values are 0: the others, each under 2^-40 of
    it, add up to less than half of fp16's smallest number, so nothing is left of them."""
    d, page, n = 128, 64, 200000
    pages = -(-n // page)
    k = torch.zeros(pages, 1, page, d, device="cuda")
    k[7, 0, 3] = 1.0
    v = torch.ones(pages, 1, page, d, device="cuda")
    v[7, 0, 3] = 0
    if held == E4M3:
        one = torch.ones(pages, 1, page, device="cuda")
        cache = rtp.PagedKVCache.from_tensors(k.to(E4M3), v.to(E4M3), one, one.clone())
    else:
        cache = rtp.PagedKVCache.from_tensors(k.to(held), v.to(held))
    q = torch.full((1, 8, d), 0.25, device="cuda", dtype=F16)              # scores: 32 and 0
    got = rtp.paged_attention(q, cache, torch.arange(pages, dtype=torch.int32, device="cuda")[None],
                              torch.tensor([n], dtype=torch.int32, device="cuda"), 1.0)
    assert n * math.exp(-32) < 2.0 ** -25 and (got == 0).all()


def test_cache_offsets_past_32_bits():
    """Rows whose element offset passes 2^31: written, read back and attended."""
    page, hk, d = 64, 8, 128
    pages = (1 << 31) // (page * hk * d) + 40
    cache = rtp.PagedKVCache(pages, page, hk, d, E4M3)
    tokens = 100
    q, k, v = _heads(31, tokens, 8, hk, d, BF16)
    rope, pos = rtp.rope_table(128, d, device="cuda"), torch.arange(tokens, device="cuda")
    w, _ = _weights(31, d, BF16)
    table = torch.tensor([[pages - 1, pages - 17]], dtype=torch.int32, device="cuda")
    slots = table[0].long()[pos // page] * page + pos % page
    rtp.qk_norm_rope_write(q, k, v, w, w, rope, pos, cache, slots, EPS)
    got = cache.read(slots, F32)
    for name, x in zip("kv", got):
        H.within(x, H.rows_of(cache, name, slots // page, slots % page), 2 * H.U32 * x.double().abs(), name)
    assert got[1].abs().sum() > 0 and cache.k_scale[:pages - 17].abs().max() == 0
    _check_attention(q[-1:].contiguous(), cache, table, torch.tensor([tokens], dtype=torch.int32, device="cuda"))
    del cache
    torch.cuda.empty_cache()


# ---- streams, graphs, devices ------------------------------------------------------------

def test_two_streams_and_two_captured_graphs():
    """Two attention calls in flight on two streams and as two graphs replayed at once share
    nothing; a captured call follows lengths that change."""
    page, hk, d = 16, 1, 128
    cache = _filled(33, 700, page, hk, d, BF16)
    qs = [_normal(_gen(34 + i), 3, 8, d).to(BF16) for i in range(2)]
    lens = [torch.tensor(n, dtype=torch.int32, device="cuda") for n in ([3000, 10, 700], [1, 4000, 0])]
    tables = [_table(33 + i, l.tolist(), page, 700, width=256) for i, l in enumerate(lens)]
    want = [rtp.paged_attention(q, cache, t, l) for q, t, l in zip(qs, tables, lens)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(rtp.paged_attention(qs[i], cache, tables[i], lens[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
    graphs, held = [], []
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            held.append(rtp.paged_attention(qs[i], cache, tables[i], lens[i]))
        graphs.append(g)
    for _ in range(10):
        for h in held:
            h.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])
    lens[0].copy_(torch.tensor([7, 4096, 0], dtype=torch.int32))
    tables[0].copy_(torch.randint(700, (3, 256), generator=_gen(40), device="cuda").to(torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0], rtp.paged_attention(qs[0], cache, tables[0], lens[0]))


@pytest.mark.parametrize("dtype,held", [(BF16, BF16), (F16, E4M3), (F32, F32)])
@pytest.mark.parametrize("longest", [300, 3000])
def test_attention_of_queries_at_odd_addresses(dtype, held, longest):
    """Queries whose elements no 4-byte load takes, and outputs given; an output that no
    vector store takes is refused."""
    page, d, lens = 16, 64, [longest, 1, 17]
    cache = _filled(29, 220, page, 1, d, held)
    table, lens_t = _table(29, lens, page, 220), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = _normal(_gen(29), 3, 9, d + 1).to(dtype)[:, 1:, 1:]
    want, _ = _check_attention(q, cache, table, lens_t)
    room = torch.full((3 * 8 * d + 16,), 5.0, dtype=dtype, device="cuda")
    out = room[8:-8].view(3, 8, d)
    assert rtp.paged_attention(q, cache, table, lens_t, out=out) is out and torch.equal(out, want)
    assert (room[:8] == 5).all() and (room[-8:] == 5).all()
    with pytest.raises(rtp.RMSNormTPError, match="aligned"):
        rtp.paged_attention(q, cache, table, lens_t, out=room[1:3 * 8 * d + 1].view(3, 8, d))


def test_results_do_not_depend_on_dependent_launch():
    page, d = 16, 128
    cache = _filled(30, 300, page, 2, d, BF16)
    lens_t = torch.tensor([4000, 0, 3, 700], dtype=torch.int32, device="cuda")
    table = _table(30, lens_t.tolist(), page, 300)
    q, k, v = _heads(30, 4, 8, 2, d, BF16)
    w, _ = _weights(30, d, BF16)
    rope, pos = rtp.rope_table(64, d, device="cuda"), _positions(30, 4, 64)
    dq, dk, _ = _heads(32, 4, 8, 2, d, BF16, "own")

    def all_of_them():
        a, b = rtp.qk_norm_rope(q, k, w, w, rope, pos)
        out = rtp.paged_attention(a, cache, table, lens_t, return_lse=True)
        return [a, b, *out, *rtp.qk_norm_rope_backward(dq, dk, q, k, w, w, rope, pos)]

    want = all_of_them()
    rtp.set_dependent_launch(False)
    try:
        for a, b in zip(want, all_of_them()):
            assert torch.equal(a, b)
    finally:
        rtp.set_dependent_launch(True)


def test_first_calls_inside_a_capture():
    """A process whose first call of each operator is captured (its kernels are loaded and
    their shared-memory limits raised during the capture)."""
    code = """
import torch, rmsnorm_tp_b200 as rtp
g = torch.Generator(device="cuda").manual_seed(1)
q, k, v = (torch.randn(5, n, 128, generator=g, device="cuda").bfloat16() for n in (8, 2, 2))
w = torch.ones(128, device="cuda").bfloat16()
rope, pos = rtp.rope_table(64, 128, device="cuda"), torch.arange(5, device="cuda")
cache = rtp.PagedKVCache(64, 16, 2, 128, torch.float8_e4m3fn)
slots = torch.arange(5, device="cuda") * 3
table = torch.arange(60, dtype=torch.int32, device="cuda").expand(5, 60)
lens = torch.tensor([13, 900, 0, 5, 1], dtype=torch.int32, device="cuda")
def run():
    a = rtp.qk_norm_rope_write(q, k, v, w, w, rope, pos, cache, slots)
    return [a, *rtp.paged_attention(a, cache, table, lens, return_lse=True), *cache.read(slots),
            *rtp.qk_norm_rope(q, k, w, w, rope, pos), *rtp.qk_norm_rope_backward(q, k, q, k, w, w, rope, pos)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    held = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(held, run()))
"""
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]


def test_captured_turn_write_read_and_backward():
    tokens, hq, hk, d = 40, 8, 2, 128
    q, k, v = _heads(35, tokens, hq, hk, d, BF16)
    dq, dk, _ = _heads(36, tokens, hq, hk, d, BF16, "own")
    qw, kw = _weights(35, d, BF16)
    rope, pos = rtp.rope_table(256, d, device="cuda"), _positions(35, tokens, 256)
    cache, slots = rtp.PagedKVCache(4, 16, hk, d, E4M3), torch.arange(tokens, device="cuda")

    def all_of_them():
        return [*rtp.qk_norm_rope(q, k, qw, kw, rope, pos), *rtp.qk_norm_rope_backward(dq, dk, q, k, qw, kw, rope, pos),
                rtp.qk_norm_rope_write(q, k, v, qw, kw, rope, pos, cache, slots), *cache.read(slots, F32)]

    # an eager graph of the same leaves lives while the backward is captured
    leaf = q.clone().requires_grad_()
    alive = rtp.qk_norm_rope_with_grad(leaf, k.clone(), qw, kw, rope, pos.clone())
    all_of_them()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = all_of_them()
    q.copy_(_normal(_gen(37), tokens, hq, d).to(BF16))
    pos.copy_(_positions(38, tokens, 256))
    slots.copy_(torch.randperm(64, generator=_gen(39), device="cuda")[:tokens])
    g.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in held]
    for a, b in zip(got, all_of_them()):
        assert torch.equal(a, b)
    alive[0].sum().backward()
    assert leaf.grad is not None


def test_python_surface_refuses():
    q, k, v = _heads(41, 4, 4, 2, 64, BF16, "own")
    w, _ = _weights(41, 64, BF16)
    rope, pos = rtp.rope_table(16, 64, device="cuda"), torch.arange(4, device="cuda")
    cache = rtp.PagedKVCache(2, 16, 2, 64)
    slots = torch.arange(4, device="cuda")
    for bad in (dict(k=k.float()), dict(k=k[:3]), dict(k=k[..., :32]), dict(q=q.double()), dict(qw=None), dict(qw=w.float()),
                dict(qw=w[:32]), dict(rope=rope.double()), dict(rope=rope[:, :63]), dict(pos=pos.int()), dict(pos=pos[:3]),
                dict(q=q.transpose(1, 2)), dict(pos=pos.cpu())):
        a = {**dict(q=q, k=k, qw=w, kw=w, rope=rope, pos=pos), **bad}
        with pytest.raises(AssertionError):
            rtp.qk_norm_rope(a["q"], a["k"], a["qw"], a["kw"], a["rope"], a["pos"])
    for outs in ((q.float(), None), (q[:, :2], None), (None, q)):
        with pytest.raises(AssertionError):
            rtp.qk_norm_rope(q, k, w, w, rope, pos, q_out=outs[0], k_out=outs[1])
    with pytest.raises(rtp.RMSNormTPError, match="overlaps"):
        rtp.qk_norm_rope(q, q[:, :2], w, w, rope, pos, q_out=q)
    with pytest.raises(rtp.RMSNormTPError, match="overlap one another"):
        rtp.qk_norm_rope(q, k, w, w, rope, pos, q_out=q[:1].clone().expand(4, -1, -1))
    for bad in (dict(v=v[:, :1]), dict(slots=slots.int()), dict(cache=rtp.PagedKVCache(2, 16, 1, 64)),
                dict(cache=rtp.PagedKVCache(2, 16, 2, 64, F16)), dict(cache=rtp.PagedKVCache(2, 16, 2, 128))):
        a = {**dict(v=v, cache=cache, slots=slots), **bad}
        with pytest.raises(AssertionError):
            rtp.qk_norm_rope_write(q, k, a["v"], w, w, rope, pos, a["cache"], a["slots"])
    for bad in ((q.float(), cache), (q[:, :3], cache), (q[..., :32], cache)):
        with pytest.raises(AssertionError):
            rtp.paged_attention(*bad, torch.zeros(4, 2, dtype=torch.int32, device="cuda"),
                                torch.zeros(4, dtype=torch.int32, device="cuda"))
    for table, lens in ((torch.zeros(4, 2, dtype=torch.int64, device="cuda"), pos.int()),
                        (torch.zeros(3, 2, dtype=torch.int32, device="cuda"), pos.int()),
                        (torch.zeros(4, 2, dtype=torch.int32, device="cuda"), pos),
                        (torch.zeros(2, 4, dtype=torch.int32, device="cuda").t(), pos.int())):
        with pytest.raises(AssertionError):
            rtp.paged_attention(q, cache, table, lens)
    with pytest.raises(AssertionError):
        rtp.paged_attention(q, cache, torch.zeros(4, 2, dtype=torch.int32, device="cuda"), pos.int(), out=q[:, :2])
    for bad in (dict(dtype=torch.int8), dict(head_dim=24), dict(head_dim=272), dict(num_pages=0), dict(page_size=0)):
        with pytest.raises(AssertionError):
            rtp.PagedKVCache(**{**dict(num_pages=2, page_size=16, num_kv_heads=1, head_dim=64), **bad})
    with pytest.raises(AssertionError):
        rtp.PagedKVCache.from_tensors(cache.k, cache.v, k_scale=rope)
    with pytest.raises(AttributeError):
        cache.k = cache.v
    with pytest.raises(AssertionError):
        cache.read(slots.int())
    with pytest.raises(AssertionError):
        cache.read(slots, torch.int8)


# ---- together ----------------------------------------------------------------------------

@pytest.mark.parametrize("held", [BF16, E4M3])
def test_decode_between_the_norms(held):
    """A prefill written into the cache, then decode steps as a block runs them at TP = 1:
    norm of the residual stream, projection, head norms + rotation + cache write, attention,
    and the row-parallel linear that adds the residual and norms again. The attention half is
    checked against the 64-bit formulas at each step from the step's own inputs."""
    hidden, hq, hk, d, page = 512, 4, 2, 128, 16
    batch, prompt, steps = 3, 37, 4
    g = _gen(51)
    w_qkv = (_normal(g, (hq + 2 * hk) * d, hidden) * hidden ** -0.5).to(BF16)
    w_o = (_normal(g, hidden, hq * d) * (hq * d) ** -0.5).to(BF16)
    qw, kw = _weights(51, d, BF16)
    norm_w = (1 + 0.1 * _normal(g, hidden)).to(BF16)
    rope = rtp.rope_table(128, d, device="cuda")
    cache = rtp.PagedKVCache(32, page, hk, d, held)
    table = torch.randperm(32, generator=g, device="cuda")[:batch * 8].view(batch, 8).to(torch.int32)
    slot_of = lambda seq, pos: table[seq, pos // page].long() * page + pos % page  # noqa: E731
    norm = rtp.FusedTPRMSNorm(hidden, eps=EPS)
    out_proj = rtp.FusedTPLinearRMSNorm(hidden, eps=EPS, num_max_rows=128)
    try:
        split = lambda x: (t.unflatten(1, (-1, d)) for t in (x @ w_qkv.t()).split([hq * d, hk * d, hk * d], 1))  # noqa: E731
        seq = torch.arange(batch, device="cuda").repeat_interleave(prompt)
        pos = torch.arange(prompt, device="cuda").repeat(batch)
        x = norm.forward(_normal(g, batch * prompt, hidden).to(BF16), norm_w)
        rtp.qk_norm_rope_write(*split(x), qw, kw, rope, pos, cache, slot_of(seq, pos), EPS)
        stream = _normal(g, batch, hidden).to(BF16)
        x = norm.forward(stream, norm_w)
        lens = torch.full((batch,), prompt, dtype=torch.int32, device="cuda")
        for step in range(steps):
            q, k, v = split(x)
            pos = lens.long()
            slots = slot_of(torch.arange(batch, device="cuda"), pos)
            q_out = rtp.qk_norm_rope_write(q, k, v, qw, kw, rope, pos, cache, slots, EPS)
            lens = lens + 1
            H.within(q_out, *H.forward(q, qw, rope, pos, EPS, False), "q")
            want_k, slop = H.forward(k, kw, rope, pos, EPS, False)
            if held == E4M3:
                H.within_e4m3(cache.k.view(torch.uint8)[slots // page, :, slots % page].view(E4M3),
                              cache.k_scale[slots // page, :, slots % page], want_k, slop, "k")
            else:
                H.within(cache.k[slots // page, :, slots % page], want_k, slop, "k")
            a, _ = _check_attention(q_out, cache, table, lens)
            before = stream.clone()
            x = out_proj.forward(a.flatten(1), w_o, norm_w, residual=stream)
            z = before.double() + a.flatten(1).double() @ w_o.double().t()
            # two roundings to bf16 (the linear's sum, the residual's) of at most 2^-8 each
            assert ((stream.double() - z).abs() <= 2 ** -8 * (z.abs() + (z - before.double()).abs()) * 1.01 + 2e-4).all()
    finally:
        norm.destroy()
        out_proj.destroy()
