"""The operators on query / key heads, the paged cache and the single-token attention
in 64 bits, written from their formulas, with the bounds their outputs are held to.

Bounds. A rounding to type t is off by at most finfo(t).eps / 2 of the value (and half
the smallest subnormal). fp32 arithmetic before it: a sum of n terms by at most
n * 2^-24 of the sum of their magnitudes, each other operation by 2^-24 of its result
(rsqrtf, exp2f, log2f: 2 ulp, counted as four such)."""
import torch

U32 = 2.0 ** -24
E4M3_MAX, E4M3_FLOOR = 448.0, 2.0 ** -100
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def turn(x, rope, positions, interleaved, back=False):
    """R(p) x of [tokens, heads, dim] (back: its transpose), and the sum of the magnitudes
    of each element's two terms."""
    table = rope.double()[positions.clamp(0, rope.shape[0] - 1)]
    bad = (positions < 0) | (positions >= rope.shape[0])
    table = table.masked_fill(bad[:, None], float("nan"))
    half = rope.shape[1] // 2
    c, s = table[:, None, :half], table[:, None, half:]
    s = -s if back else s
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y, size = x.clone(), x.abs()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, size


def norm(x, w, eps):
    inv = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    return x * inv * w, inv


def forward(x, w, rope, positions, eps, interleaved):
    """(y in 64 bits, bound of the fp32 arithmetic)."""
    x = x.double()
    if w is not None:
        x, _ = norm(x, w.double(), eps)
    y, size = turn(x, rope, positions, interleaved)
    # the sum of squares (half of its relative error reaches the root), two products of the
    # norm, and the turn's two products and sum
    return y, (x.shape[-1] / 2 + 16) * U32 * size


def backward(dy, x, w, rope, positions, eps, interleaved):
    """(dx, its bound, dw, its bound)."""
    g, size = turn(dy.double(), rope, positions, interleaved, back=True)
    if w is None:
        return g, 8 * U32 * size, None, None
    x, w = x.double(), w.double()
    d = x.shape[-1]
    _, inv = norm(x, w, eps)
    along = (g * w * x).mean(-1, keepdim=True)
    dx = inv * g * w - x * inv.pow(3) * along
    most = inv * size * w.abs() + x.abs() * inv.pow(3) * (size * w.abs() * x.abs()).mean(-1, keepdim=True)
    n = x.shape[0] * x.shape[1]
    dw = (g * x * inv).sum((0, 1))
    sw = (size * x.abs() * inv).sum((0, 1))
    return dx, (2 * d + 24) * U32 * most, dw, (n + d / 2 + 24) * U32 * sw


def within(got, want, slop, what):
    """`got` (of its type) within its rounding and `slop` of `want`; NaN exactly where it has NaN."""
    dtype = got.dtype
    got = got.double()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    fine = ~torch.isnan(want)
    bound = half_step(dtype) * (want.abs() + slop) + slop + SMALLEST[dtype] / 2
    over = ((got - want).abs() - bound)[fine]
    assert over.numel() == 0 or over.max() <= 0, \
        f"{what}: {int((over > 0).sum())} of {over.numel()} off, worst by {over.max().item():.3g}"


def within_e4m3(codes, scale, want, slop, what):
    """An e4m3 row against the values it stands for: the code is a rounding of value /
    scale (half a step 2^-4, or half the smallest subnormal 2^-9), the scale amax / 448."""
    most = want.abs().amax(-1, keepdim=True).clamp(min=E4M3_FLOOR)
    loose = slop.amax(-1, keepdim=True)
    s = scale.double()[..., None]
    assert ((s - most / E4M3_MAX).abs() <= loose / E4M3_MAX + 4 * U32 * s).all(), f"{what}: scales"
    ratio = want / s
    bound = torch.maximum(2.0 ** -4 * ratio.abs(), torch.tensor(2.0 ** -10, device=want.device)) * (1 + 2.0 ** -10)
    over = (codes.double() - ratio).abs() - bound - 1.1 * (slop + loose + 8 * U32 * want.abs()) / s
    assert over.max() <= 0, f"{what}: codes off by {over.max().item():.3g} beyond the bound"


def rows_of(cache, name, pages, offsets):
    """Rows [count, kv_heads, dim] in 64 bits as the cache holds them."""
    x = getattr(cache, name)
    scale = getattr(cache, name + "_scale")
    if scale is None:
        return x[pages, :, offsets].double()
    return x.view(torch.uint8)[pages, :, offsets].view(x.dtype).double() * scale[pages, :, offsets].double()[..., None]


def attend(q, cache, page_table, seq_lens, scale, p_step):
    """(out, its slop, lse, its slop). `p_step`: half step of the type the kernel rounds
    the softmax's numerators to."""
    batch, hq, d = q.shape
    page, hk = cache.page_size, cache.num_kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((batch, hq), float("-inf"), dtype=torch.float64, device=q.device)
    slop, lslop = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(batch):
        n = min(max(int(seq_lens[b]), 0), page_table.shape[1] * page)
        t = torch.arange(n, device=q.device)
        pages = page_table[b].long()[t // page] if n else t
        live = (pages >= 0) & (pages < cache.num_pages)
        pages, off = pages[live], (t % page)[live]
        if not pages.numel():
            continue
        k, v = (rows_of(cache, m, pages, off).transpose(0, 1).repeat_interleave(hq // hk, 0) for m in ("k", "v"))
        x = q[b].double()
        s = torch.einsum("hd,hnd->hn", x, k) * scale
        size = torch.einsum("hd,hnd->hn", x.abs(), k.abs()).nan_to_num(posinf=0.0) * abs(scale)
        m = s.amax(-1, keepdim=True)
        ref = torch.where(torch.isneginf(m), 0.0, m)
        p = torch.exp(s - ref)
        l = p.sum(-1, keepdim=True)
        out[b] = torch.where(l == 0, 0.0, torch.einsum("hn,hnd->hd", p, v) / l)
        lse[b] = (ref + torch.log(l)).squeeze(-1)
        # a score is off by its sum's error and by its own rounding and the maximum's; every p
        # relatively by twice that (its own and the maximum's), the numerators by p_step more
        e = (((d + 8) * U32 * size).amax(-1) + 16 * U32 * s.abs().nan_to_num(posinf=0, neginf=0).amax(-1))
        n = pages.numel()
        rel = 2 * e + (2 * n + 64) * U32 + p_step
        around = torch.einsum("hn,hnd->hd", p, v.abs()) / l.clamp(min=1e-300)
        # numerators under the 16-bit type's smallest number are lost: 2^-25 of the largest
        lost = 2.0 ** -25 * n * v.abs().amax(1) / l.clamp(min=1e-300) if p_step > 2.0 ** -20 else 0.0
        slop[b] = (rel[:, None] * around + lost).nan_to_num()
        lslop[b] = e + (n + 64) * U32 + 8 * U32 * lse[b].abs().nan_to_num(neginf=0.0)
    return out, slop, lse, lslop
