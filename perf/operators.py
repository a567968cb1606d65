"""Work of the attention operators: what is measured, in plain form and through the package.

Four kinds of case, over one set of operators:
  "turn"    norms of query and key heads with the position rotation
  "grad"    the backward pass of "turn"
  "write"   "turn", with K and V written into a paged cache (16-bit, or e4m3 codes with a scale
            for each token and head)
  "read"    cache rows brought back by slot
  "attend"  attention of one new token for each sequence over the paged cache
"""
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}
_EPS = 1e-6
_LARGEST = 448.0        # of e4m3
_FLOOR = 2.0 ** -100    # smallest row maximum that a scale is made of


# ---- cases -------------------------------------------------------------------

def _turn_case(do, tokens, hq, hk, d, r, dtype, inter=False, norm=True, span=0, **more):
    return dict(do=do, tokens=tokens, q_heads=hq, kv_heads=hk, head_dim=d, rotary=r, dtype=dtype,
                interleaved=inter, norm=norm, span=span, **more)


def listed():
    return [
        # one decode step of a few sequences, 4096-wide model: latency
        dict(_turn_case("turn", 8, 32, 8, 128, 128, "bf16"), name="turn_decode"),
        # a prefill of four prompts of 2048 tokens, the same heads
        dict(_turn_case("turn", 8192, 32, 8, 128, 128, "bf16", span=2048), name="turn_prefill"),
        # part of each head rotated, neighbouring pairs, full precision, odd sizes
        dict(_turn_case("turn", 1531, 12, 3, 80, 32, "f32", inter=True, span=511), name="turn_partial"),
        # a training step's backward over 8192 tokens
        dict(_turn_case("grad", 8192, 32, 8, 128, 128, "bf16", span=4096), name="grad_train"),
        # a small odd micro-batch on one rank of a tensor-parallel group, fp16
        dict(_turn_case("grad", 333, 8, 1, 64, 64, "f16", span=333), name="grad_small"),
        # a decode batch on one rank of eight (8192-wide model): one kv head, e4m3 cache
        dict(_turn_case("write", 64, 8, 1, 128, 128, "bf16", cache="e4m3", page=64), name="write_decode"),
        # a prefill written into an e4m3 cache
        dict(_turn_case("write", 8192, 32, 8, 128, 128, "bf16", span=2048, cache="e4m3", page=64),
             name="write_prefill"),
        # a cached prefix of 32768 tokens brought back for a prefill that continues it
        dict(do="read", tokens=32768, kv_heads=8, head_dim=128, dtype="bf16", cache="e4m3", page=64,
             name="read_prefix"),
        # one long sequence on one rank of eight: work has to come from the length alone
        dict(do="attend", batch=1, longest=262144, q_heads=8, kv_heads=1, head_dim=128, dtype="bf16",
             cache="bf16", page=64, name="attend_long"),
        # a ragged serving batch over an e4m3 cache
        dict(do="attend", batch=64, longest=16384, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16",
             cache="e4m3", page=64, name="attend_batch"),
        # every query head with its own key head, small pages, fp16
        dict(do="attend", batch=48, longest=2011, q_heads=16, kv_heads=16, head_dim=64, dtype="f16",
             cache="f16", page=16, name="attend_heads"),
        # a few short chats on one rank of eight: latency
        dict(do="attend", batch=4, longest=700, q_heads=8, kv_heads=1, head_dim=128, dtype="bf16",
             cache="bf16", page=16, name="attend_short"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    do = rng.choice(["turn", "grad", "write", "read", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    cache = rng.choice(["e4m3", dtype])
    page = rng.choice([16, 32, 64, 128, 48, 7])
    if do == "read":
        hk, d = rng.randint(1, 16), rng.choice([64, 96, 128, 192, 256])
        most = min(65536, (40 << 20) // (hk * d))
        return dict(do=do, tokens=_log(rng, 1, most), kv_heads=hk, head_dim=d, dtype=dtype,
                    cache=cache, page=page)
    if do == "attend":
        hk, d, group = rng.randint(1, 8), rng.choice([64, 96, 128, 192, 256]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16, 20])
        batch = _log(rng, 1, 256)
        most = max(16, min(131072, (400 << 20) // (batch * hk * d * 2)))
        return dict(do=do, batch=batch, longest=_log(rng, 1, most), q_heads=hk * group, kv_heads=hk,
                    head_dim=d, dtype=dtype, cache=cache, page=page)
    hk = rng.randint(1, 8)
    hq = hk * rng.choice([1, 2, 3, 4, 7, 8])
    if do == "write":
        d = rng.choice([64, 96, 128, 192, 256])
    else:
        d = rng.choice([32, 64, 80, 96, 128, 192, 256, 50])
        dtype = rng.choice(["bf16", "f16", "f32"])
    r = rng.choice([d, d, d // 2 // 2 * 2])
    most = min(16384, (64 << 20) // ((hq + 2 * hk) * d))
    tokens = _log(rng, 1, most)
    more = dict(cache=cache, page=page) if do == "write" else {}
    return _turn_case(do, tokens, hq, hk, d, r, dtype, inter=rng.random() < 0.3, norm=rng.random() < 0.8,
                      span=rng.choice([0, _log(rng, 1, tokens)]), **more)


def _lengths(c):
    """The sequences' lengths: one the longest, one empty, one of a single token, the others spread."""
    n, most = c["batch"], c["longest"]
    lens = [1 + int((most - 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]
    lens[n // 2] = most
    if n > 4:
        lens[1], lens[2] = 0, 1
    return lens


def _written(c):
    """Tokens of a "write" that have a slot: each seventeenth of a batch is padding."""
    return c["tokens"] - c["tokens"] // 17


def _pages(c, tokens):
    return max(1, -(-tokens // c["page"]) * 9 // 8 + 1)


def work(c):
    s = _SIZE[c["dtype"]]
    if c["do"] == "attend":
        live = sum(_lengths(c))
        row = c["head_dim"] * _SIZE[c["cache"]] + (4 if c["cache"] == "e4m3" else 0)
        head = c["head_dim"] * s
        table = sum(-(-n // c["page"]) for n in _lengths(c)) * 4 + c["batch"] * 4
        return {"bytes": 2 * live * c["kv_heads"] * row + c["batch"] * c["q_heads"] * (2 * head + 4) + table,
                "flops": 4 * live * c["q_heads"] * c["head_dim"]}
    if c["do"] == "read":
        n = c["tokens"] * c["kv_heads"]
        row = c["head_dim"] * _SIZE[c["cache"]] + (4 if c["cache"] == "e4m3" else 0)
        return {"bytes": 2 * n * (row + c["head_dim"] * s) + 8 * c["tokens"], "flops": 2 * n * c["head_dim"]}
    t, d, hq, hk = c["tokens"], c["head_dim"], c["q_heads"], c["kv_heads"]
    table = (min(t, c["span"]) if c["span"] else t) * c["rotary"] * 4 + 8 * t + (2 * d * s if c["norm"] else 0)
    if c["do"] == "turn":
        return {"bytes": 2 * t * (hq + hk) * d * s + table, "flops": 8 * t * (hq + hk) * d}
    if c["do"] == "grad":
        return {"bytes": 3 * t * (hq + hk) * d * s + table + (2 * d * s if c["norm"] else 0),
                "flops": 16 * t * (hq + hk) * d}
    row = d * _SIZE[c["cache"]] + (4 if c["cache"] == "e4m3" else 0)
    return {"bytes": (2 * t * hq + 2 * _written(c) * hk) * d * s + 2 * _written(c) * hk * row + table + 8 * t,
            "flops": 8 * t * (hq + 2 * hk) * d}


# ---- what a program has in hand ------------------------------------------------

def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    type_ = _TYPES[c["dtype"]]
    normal = lambda *n: torch.randn(*n, generator=g, device="cuda")  # noqa: E731
    state = {"do": c["do"]}
    if c["do"] in ("write", "read", "attend"):
        d, hk, page = c["head_dim"], c["kv_heads"], c["page"]
        lens = _lengths(c) if c["do"] == "attend" else [c["tokens"]]
        used = [-(-n // page) for n in lens]
        pages = _pages(c, sum(used) * page)
        order = torch.randperm(pages, generator=g, device="cuda")
        state["cache"] = _cache(c, pages, normal)
    if c["do"] == "attend":
        width = max(1, max(used))
        # one row of pages for each sequence, -1 behind its last page
        count = torch.tensor(used, device="cuda")
        at = torch.arange(width, device="cuda")
        live = at < count[:, None]
        first = torch.cumsum(count, 0) - count
        state["page_table"] = torch.where(live, order[(first[:, None] + at).clamp(max=pages - 1)], -1).to(torch.int32)
        state["seq_lens"] = torch.tensor(lens, device="cuda", dtype=torch.int32)
        # normed queries, a little sharper than unit scores
        state["q"] = (2.0 * normal(c["batch"], c["q_heads"], d)).to(type_)
        state["scale"] = d ** -0.5
        return state
    if c["do"] == "read":
        pos = torch.arange(c["tokens"], device="cuda")
        state["slots"] = order[pos // page] * page + pos % page
        state["dtype"] = type_
        return state
    t, d, hq, hk = c["tokens"], c["head_dim"], c["q_heads"], c["kv_heads"]
    # q, k and v as the projection leaves them: column blocks of one matrix, a few channels much
    # larger than the others
    loud = torch.where(torch.rand((hq + 2 * hk) * d, generator=g, device="cuda") < 0.01, 20.0, 1.0)
    qkv = (normal(t, (hq + 2 * hk) * d) * loud).to(type_)
    state["q"] = qkv[:, :hq * d].view(t, hq, d)
    state["k"] = qkv[:, hq * d:(hq + hk) * d].view(t, hk, d)
    state["v"] = qkv[:, (hq + hk) * d:].view(t, hk, d)
    weight = lambda: (1.0 + 0.1 * normal(d)).to(type_) if c["norm"] else None  # noqa: E731
    state["q_weight"], state["k_weight"] = weight(), weight()
    far = 32768
    turn = torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(0, c["rotary"], 2, device="cuda", dtype=torch.float64) / c["rotary"])
    state["rope"] = torch.cat([turn.cos(), turn.sin()], 1).float()
    if c["span"]:  # prompts of `span` tokens, one behind another
        state["positions"] = torch.arange(t, device="cuda") % c["span"]
    else:          # one new token of each sequence
        state["positions"] = torch.randint(far, (t,), generator=g, device="cuda")
    state["interleaved"] = c["interleaved"]
    if c["do"] == "grad":
        state["dq"], state["dk"] = normal(t, hq, d).to(type_), normal(t, hk, d).to(type_)
    if c["do"] == "write":
        pos = torch.arange(t, device="cuda")
        slots = order[pos // page] * page + pos % page
        state["slots"] = torch.where(pos % 17 == 16, -1, slots)
    return state


def _cache(c, pages, normal):
    """A cache in use: every page holds an earlier token's rows."""
    shape = (pages, c["kv_heads"], c["page"], c["head_dim"])
    if c["cache"] != "e4m3":
        k, v, ks, vs = normal(*shape).to(_TYPES[c["cache"]]), normal(*shape).to(_TYPES[c["cache"]]), None, None
    else:
        (k, ks), (v, vs) = _codes(normal(*shape)), _codes(normal(*shape) * normal(*shape[:3], 1).exp())
    if own:  # the package's handle of these same tensors
        import rmsnorm_tp_b200 as rtp
        return rtp.PagedKVCache.from_tensors(k, v, ks, vs)
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}


# ---- one pass --------------------------------------------------------------------

def run(s):
    do = s["do"]
    if own:
        import rmsnorm_tp_b200 as rtp
        if do == "turn":
            return rtp.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["rope"], s["positions"],
                                    eps=_EPS, interleaved=s["interleaved"])
        if do == "grad":
            return rtp.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["q_weight"], s["k_weight"],
                                             s["rope"], s["positions"], eps=_EPS, interleaved=s["interleaved"])
        if do == "write":
            c = s["cache"]
            q = rtp.qk_norm_rope_write(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["rope"],
                                       s["positions"], c, s["slots"], eps=_EPS, interleaved=s["interleaved"])
            return [q, c.k, c.v, c.k_scale, c.v_scale]
        if do == "read":
            return s["cache"].read(s["slots"], s["dtype"])
        return rtp.paged_attention(s["q"], s["cache"], s["page_table"], s["seq_lens"], scale=s["scale"],
                                   return_lse=True)
    if do == "turn":
        return _forward(s, "q").to(s["q"].dtype), _forward(s, "k").to(s["k"].dtype)
    if do == "grad":
        dq, dqw = _backward(s, "q")
        dk, dkw = _backward(s, "k")
        return dq, dk, dqw, dkw
    c = s["cache"]
    if do == "write":
        _store(c, s["slots"], _forward(s, "k"), s["v"].float())
        return [_forward(s, "q").to(s["q"].dtype), c["k"], c["v"], c["k_scale"], c["v_scale"]]
    if do == "read":
        page = c["k"].shape[2]
        at, off = s["slots"] // page, s["slots"] % page
        return tuple(_rows(c, n, at, off).to(s["dtype"]) for n in ("k", "v"))
    return _attend(s)


def _sides(s):
    """cos and sin of each token, for all its heads."""
    table = s["rope"][s["positions"]][:, None, :]
    return table.chunk(2, -1)


def _turn(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    a, rest = x[..., :r], x[..., r:]
    if interleaved:
        u, v = a[..., 0::2], a[..., 1::2]
        y = torch.stack((u * cos - v * sin, u * sin + v * cos), -1).flatten(-2)
    else:
        u, v = a.chunk(2, -1)
        y = torch.cat((u * cos - v * sin, u * sin + v * cos), -1)
    return torch.cat((y, rest), -1)


def _forward(s, n):
    x, w = s[n].float(), s[n + "_weight"]
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * w.float()
    return _turn(x, *_sides(s), s["interleaved"])


def _backward(s, n):
    x, w, type_ = s[n].float(), s[n + "_weight"], s[n].dtype
    cos, sin = _sides(s)
    g = _turn(s["d" + n].float(), cos, -sin, s["interleaved"])
    if w is None:
        return g.to(type_), None
    inv = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
    gw = g * w.float()
    dx = inv * gw - x * inv ** 3 * (gw * x).mean(-1, keepdim=True)
    return dx.to(type_), (g * x * inv).sum((0, 1)).to(type_)


def _codes(x):
    """e4m3 codes of rows and each row's scale."""
    most = x.abs().amax(-1, keepdim=True).clamp(min=_FLOOR)
    return (x * (_LARGEST / most)).clamp(-_LARGEST, _LARGEST).to(torch.float8_e4m3fn), (most / _LARGEST).squeeze(-1)


def _store(c, slots, k, v):
    page = c["k"].shape[2]
    live = slots >= 0
    at, off = slots[live] // page, slots[live] % page
    for n, x in (("k", k[live]), ("v", v[live])):
        if c[n + "_scale"] is None:
            c[n][at, :, off] = x.to(c[n].dtype)
        else:
            codes, scale = _codes(x)
            c[n].view(torch.uint8)[at, :, off] = codes.view(torch.uint8)
            c[n + "_scale"][at, :, off] = scale


def _rows(c, n, at, off):
    if c[n + "_scale"] is None:
        return c[n][at, :, off].float()
    return c[n].view(torch.uint8)[at, :, off].view(torch.float8_e4m3fn).float() * c[n + "_scale"][at, :, off][..., None]


def _spread(c, n, pages):
    """The pages of each sequence behind one another, in 32 bits: [batch, kv heads, length, head_dim]."""
    x = c[n]
    if c[n + "_scale"] is None:
        x = x[pages].float()
    else:
        x = x.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * c[n + "_scale"][pages][..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(s):
    c, q, lens = s["cache"], s["q"], s["seq_lens"]
    pages = s["page_table"].clamp(min=0).long()
    k = _spread(c, "k", pages)
    b, hk, most, d = k.shape
    live = (torch.arange(most, device=q.device) < lens[:, None])[:, None, None, :]
    x = (q.float().view(b, hk, -1, d) @ k.transpose(-1, -2)) * s["scale"]
    del k
    x = x.masked_fill(~live, float("-inf"))
    top = x.amax(-1, keepdim=True)
    top = top.masked_fill(torch.isneginf(top), 0.0)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    v = _spread(c, "v", pages).masked_fill(~live.transpose(-1, -2), 0.0)
    out = torch.where(total > 0, (p @ v) / total, 0.0)
    return out.view(b, -1, d).to(q.dtype), (top + torch.log(total)).view(b, -1)


# ---- the definition in 64 bits -----------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    if c["do"] == "read":
        return tuple(_whole(s["cache"], n).flatten(1, 2)[:, s["slots"]].transpose(0, 1) for n in ("k", "v"))
    if c["do"] == "attend":
        return _exact_attend(c, s)
    angle = s["rope"].double()[s["positions"]]
    half = angle.shape[1] // 2
    z = torch.complex(angle[:, :half], angle[:, half:])[:, None]
    if c["do"] == "grad":
        out = [_exact_grad(s, z, n) for n in ("q", "k")]
        return [out[0][0], out[1][0], out[0][1], out[1][1]]
    q, k = _exact_turn(s, z, "q"), _exact_turn(s, z, "k")
    if c["do"] == "turn":
        return q, k
    cache, got = s["cache"], [q]
    scales = []
    for n, x in (("k", k), ("v", s["v"].double())):
        held = _by_slot(_tensor(cache, n).double())   # what the pages held, by slot
        live = (s["slots"] >= 0).nonzero().flatten()
        if c["cache"] == "e4m3":
            scale = x.abs().amax(-1).clamp(min=_FLOOR) / _LARGEST
            x = x / scale[..., None]
            by = _by_slot(_tensor(cache, n + "_scale").double()[..., None])
            by[s["slots"][live]] = scale[live][..., None]
            scales.append(_by_page(by, cache, n).squeeze(-1))
        held[s["slots"][live]] = x[live]
        got.append(_by_page(held, cache, n))
    return got + (scales or [None, None])


def _tensor(cache, n):
    return cache[n] if isinstance(cache, dict) else getattr(cache, n)


def _by_slot(x):
    return x.permute(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3]).contiguous()


def _by_page(x, cache, n):
    pages, heads, page, _ = _tensor(cache, n).shape
    return x.view(pages, page, heads, -1).permute(0, 2, 1, 3)


def _whole(cache, n):
    """All rows of the cache: [kv heads, pages, page, head_dim]."""
    x, scale = _tensor(cache, n).double(), _tensor(cache, n + "_scale")
    return (x if scale is None else x * scale.double()[..., None]).transpose(0, 1)


def _spun(x, z, interleaved):
    """x with its first pairs multiplied, as complex numbers, by z."""
    half = z.shape[-1]
    y = x.clone()
    i = 2 * torch.arange(half, device=x.device) if interleaved else torch.arange(half, device=x.device)
    j = i + 1 if interleaved else i + half
    w = torch.complex(x[..., i], x[..., j]) * z
    y[..., i], y[..., j] = w.real, w.imag
    return y


def _exact_turn(s, z, n):
    x, w = s[n].double(), s[n + "_weight"]
    if w is not None:
        x = w.double() * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt()
    return _spun(x, z, s["interleaved"])


def _exact_grad(s, z, n):
    x, w = s[n].double(), s[n + "_weight"]
    g = _spun(s["d" + n].double(), z.conj(), s["interleaved"])
    if w is None:
        return g, None
    root = (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt()
    unit = x / root
    along = g * w.double()
    return ((along - unit * (along * unit).sum(-1, keepdim=True) / x.shape[-1]) / root,
            torch.einsum("thd,thd->d", g, unit))


def _exact_attend(c, s):
    lens = _lengths(c)
    if sum(lens) * c["kv_heads"] * c["head_dim"] > 1 << 30:
        return None
    group = c["q_heads"] // c["kv_heads"]
    cache = s["cache"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], float("-inf"), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if not n:
            continue
        pages = s["page_table"][b, :-(-n // c["page"])].long()
        rows = []
        for name in ("k", "v"):
            x, scale = _tensor(cache, name), _tensor(cache, name + "_scale")
            x = x.view(torch.uint8)[pages].view(x.dtype).double() if scale is not None else x[pages].double()
            x = x if scale is None else x * scale[pages].double()[..., None]
            rows.append(x.permute(1, 0, 2, 3).flatten(1, 2)[:, :n].repeat_interleave(group, 0))
        score = torch.einsum("hd,hnd->hn", s["q"][b].double(), rows[0]) * s["scale"]
        lse[b] = torch.logsumexp(score, -1)
        out[b] = torch.einsum("hn,hnd->hd", torch.softmax(score, -1), rows[1])
    return out, lse


if __name__ == "__main__":
    rng = random.Random(0)
    for case in listed() + [draw(rng) for _ in range(12)]:
        print(case, work(case))
