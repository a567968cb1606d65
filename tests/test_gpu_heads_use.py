"""Ways to use the operators on heads beside the plain call: copied and stored caches, layouts
of the projection, operands that share memory."""
import copy
import io

import pytest
import torch

import heads_oracle as H
import rmsnorm_tp_b200 as rtp

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def _normal(seed, *n):
    return torch.randn(*n, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _stored(cache):
    buf = io.BytesIO()
    torch.save(cache, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)


@pytest.mark.parametrize("held", [BF16, E4M3])
@pytest.mark.parametrize("how", [copy.deepcopy, _stored])
def test_copies_of_a_cache_are_caches_of_their_own(how, held):
    tokens, d = 20, 64
    rope, pos = rtp.rope_table(64, d, device="cuda"), torch.arange(tokens, device="cuda")
    cache = rtp.PagedKVCache(4, 16, 2, d, held)
    rows = [_normal(i, tokens, 2, d).to(BF16) for i in range(2)]
    rtp.qk_norm_rope_write(rows[0], rows[0], rows[0], None, None, rope, pos, cache, pos)
    before = [t.clone() for t in cache.read(pos)]
    cache.note = "kept"
    other = how(cache)
    assert other.note == "kept" and other.k.data_ptr() != cache.k.data_ptr() and other.dtype == held
    for a, b in zip(other.read(pos), before):
        assert torch.equal(a, b)
    rtp.qk_norm_rope_write(rows[1], rows[1], rows[1], None, None, rope, pos, other, pos)
    for a, b in zip(cache.read(pos), before):                    # the first as it was
        assert torch.equal(a, b)
    table, lens = torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.tensor([tokens], dtype=torch.int32, device="cuda")
    want = [rtp.paged_attention(rows[1][-1:], c, table, lens) for c in (cache, other)]
    assert not torch.equal(*want)
    del cache
    torch.cuda.empty_cache()
    assert torch.equal(rtp.paged_attention(rows[1][-1:], other, table, lens), want[1])


def test_a_shallow_copy_shares_the_tensors():
    cache = rtp.PagedKVCache(2, 16, 1, 64)
    other = copy.copy(cache)
    assert other.k is cache.k and other._address != cache._address


def test_write_refuses_shared_memory_and_cached_keys_turn_in_place():
    tokens, d, page = 16, 64, 16
    rope, pos = rtp.rope_table(64, d, device="cuda"), torch.arange(tokens, device="cuda") + 5
    cache = rtp.PagedKVCache.from_tensors(_normal(3, 3, 2, page, d).to(BF16), _normal(4, 3, 2, page, d).to(BF16))
    q, v = _normal(5, tokens, 4, d).to(BF16), _normal(6, tokens, 2, d).to(BF16)
    row = cache.k[1].transpose(0, 1)                             # a page's keys, [tokens, heads, d]
    for bad in ((q, row, v), (q, v, row), (cache.k.view(-1, 4, d)[:tokens], v, v)):
        with pytest.raises(rtp.RMSNormTPError, match="overlaps the cache"):
            rtp.qk_norm_rope_write(*bad, None, None, rope, pos, cache, pos)
    one = rtp.PagedKVCache.from_tensors(cache.k, cache.k)        # keys that are the values: to read
    with pytest.raises(AssertionError, match="share memory"):
        rtp.qk_norm_rope_write(q, v, v, None, None, rope, pos, one, pos)
    for a, b in zip(one.read(pos), (cache.read(pos)[0],) * 2):
        assert torch.equal(a, b)
    codes, scale = torch.zeros(2, 1, 1, 16, d, device="cuda").to(E4M3), torch.ones(1, 1, 16, device="cuda")
    with pytest.raises(AssertionError, match="share memory"):
        rtp.qk_norm_rope_write(q[:, :1], v[:, :1], v[:, :1], None, None, rope, pos,
                               rtp.PagedKVCache.from_tensors(codes[0], codes[1], scale, scale), pos)
    want = H.forward(row.clone(), None, rope, pos, 1e-6, False)
    before = cache.k.clone()
    rtp.qk_norm_rope(q, row, None, None, rope, pos, k_out=row)
    H.within(cache.k[1].transpose(0, 1), *want, "keys turned in place")
    assert torch.equal(cache.k[0], before[0]) and torch.equal(cache.k[2], before[2])


@pytest.mark.parametrize("d,r", [(128, 128), (96, 32), (50, 20)])
@pytest.mark.parametrize("tokens", [1, 77])
def test_turned_in_place_where_q_k_and_v_of_a_head_lie_side_by_side(tokens, d, r):
    heads = 5
    qkv = _normal(7, tokens, heads, 3, d).to(BF16)
    q, k, v = qkv.unbind(2)
    w = [(1 + 0.2 * _normal(8 + i, d)).to(BF16) for i in range(2)]
    rope, pos = rtp.rope_table(128, r, device="cuda"), torch.arange(tokens, device="cuda")
    want, v0 = rtp.qk_norm_rope(q, k, *w, rope, pos), v.clone()
    cache = rtp.PagedKVCache(8, 16, heads, d, BF16) if d % 16 == 0 else None
    rtp.qk_norm_rope(q, k, *w, rope, pos, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, v0)
    if cache is not None:
        want, held = rtp.qk_norm_rope(q, k, *w, rope, pos), k.clone()
        rtp.qk_norm_rope_write(q, k, v, *w, rope, pos, cache, pos, q_out=q)
        assert torch.equal(q, want[0]) and torch.equal(k, held) and torch.equal(v, v0)
        for a, b in zip(cache.read(pos), (want[1], v0)):
            assert torch.equal(a, b)


def test_a_table_that_wants_a_gradient_is_refused():
    q = _normal(9, 3, 2, 64).requires_grad_()
    rope, pos = rtp.rope_table(8, 64, device="cuda").requires_grad_(), torch.arange(3, device="cuda")
    with pytest.raises(AssertionError, match="rope"):
        rtp.qk_norm_rope_with_grad(q, q, None, None, rope, pos)
    with torch.no_grad():
        rtp.qk_norm_rope_with_grad(q, q, None, None, rope, pos)
    rtp.qk_norm_rope_with_grad(q, q, None, None, rope.detach(), pos)[0].sum().backward()
    assert q.grad is not None and rope.grad is None


@pytest.mark.parametrize("shape", [(2, 0, 16, 64), (2, 1, 0, 64)])
def test_a_cache_without_heads_or_rows_is_refused(shape):
    with pytest.raises(AssertionError, match="positive"):
        rtp.PagedKVCache.from_tensors(*(torch.zeros(shape, device="cuda") for _ in range(2)))
