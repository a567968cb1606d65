"""Operands of the operators on heads that share memory, as the C entry points judge them
(without a GPU: accepted calls end at a device that does not exist)."""
import random

import pytest

from rmsnorm_tp_b200 import _lib
from test_heads_host import KO, L, Q, QO, SLOTS, V, _cache, _forward, _rope

CK, CV, KS, VS = 0xD0000000, 0xE0000000, 0xF0000000, 0xF8000000
CACHE_BYTES = 4 * 16 * 2 * 64                # elements of k, and of v


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("name", ["q", "k", "v", "qo"])
def test_write_refuses_operands_inside_the_cache(name, e4m3):
    size = CACHE_BYTES * (1 if e4m3 else 2)
    keep, at = _cache(dtype=_lib.KV_E4M3 if e4m3 else _lib.BF16, ks=KS if e4m3 else 0, vs=VS if e4m3 else 0)
    call = lambda **kw: L.rmsnorm_qk_rope_write(_rope(**{**dict(v=V, slots=SLOTS, cache=at, ko=0), **kw}), None)  # noqa: E731
    assert call() == _lib.ERR_CUDA
    own = 8 * (4 if name in ("q", "qo") else 2) * 64 * 2          # bytes of the operand
    for start, n in [(CK, size), (CV, size)] + ([(KS, CACHE_BYTES // 64 * 4), (VS, CACHE_BYTES // 64 * 4)] if e4m3 else []):
        for inside in (start, start + n - 16, start - own + 16):
            assert call(**{name: inside}) == _lib.ERR_INVALID, hex(inside)
            assert "overlaps the cache" in _lib.last_error()
        for beside in (start + n, start - own):
            assert call(**{name: beside}) == _lib.ERR_CUDA, hex(beside)


def test_write_refuses_a_cache_whose_keys_are_its_values():
    for v in (CK, CK + 2 * CACHE_BYTES - 16):
        keep, at = _cache(v=v)
        assert L.rmsnorm_qk_rope_write(_rope(v=V, slots=SLOTS, cache=at, ko=0), None) == _lib.ERR_INVALID
        assert "k overlaps its v" in _lib.last_error()
    keep, at = _cache(v=CK + 2 * CACHE_BYTES)
    assert L.rmsnorm_qk_rope_write(_rope(v=V, slots=SLOTS, cache=at, ko=0), None) == _lib.ERR_CUDA


# q, k and v of a head side by side: [tokens, heads, 3, 64] of 16-bit elements
BETWEEN = dict(hq=4, hk=4, q=Q, k=Q + 128, qo=Q, ko=Q + 128,
               **{n: (4 * 192, 192) for n in ("qs", "ks", "qos", "kos")})


@pytest.mark.parametrize("kw", [dict(), dict(tokens=1), dict(ko=KO, kos=(256, 64)), dict(ko=Q + 256), dict(qo=QO),
                                dict(qs=(192, 1024 * 192), ks=(192, 1024 * 192), qos=(192, 1024 * 192), kos=(192, 1024 * 192))])
def test_heads_between_one_another_are_turned_in_place(kw):
    assert _forward(**{**BETWEEN, **kw}) == _lib.ERR_CUDA, _lib.last_error()


@pytest.mark.parametrize("kw", [dict(ko=Q + 64), dict(ko=Q + 320), dict(k=Q + 64, ko=KO), dict(ko=Q + 384), dict(qo=Q + 128),
                                dict(kos=(4 * 192 + 64, 192)), dict(ks=(4 * 192, 128)), dict(k=Q + 768 * 2)])
def test_heads_that_overlap_one_another_are_refused(kw):
    assert _forward(**{**BETWEEN, **kw}) == _lib.ERR_INVALID
    assert "overlap" in _lib.last_error()


def test_no_views_that_share_an_element_are_taken():
    """Random small views of q, k and their outputs around one address: a call that is taken has
    outputs that share no element with one another or with an input but their own, row for row."""
    rng = random.Random(5)
    taken = refused = 0
    for _ in range(20000):
        d, tokens, hq, hk = 2 * rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 4)
        unit = d * rng.choice([1, 1, 2, 3])
        strides = [unit, unit * hq, unit * 3, unit * tokens, 3 * unit * max(hq, hk), d + 1, rng.randint(0, 40)]
        if rng.random() < 0.6:                              # views of one matrix
            one = (rng.choice(strides), rng.choice(strides))
            st = [one] * 4
        else:
            st = [(rng.choice(strides), rng.choice(strides)) for _ in range(4)]
        at = [Q + 4 * d * rng.randint(0, 12) + 4 * rng.choice([0, 0, 0, 1]) for _ in range(2)]
        at += [at[i] if rng.random() < 0.5 else Q + 4 * d * rng.randint(0, 40) for i in range(2)]
        rc = _forward(d=d, r=d, tokens=tokens, hq=hq, hk=hk, dtype=_lib.F32, q=at[0], k=at[1], qo=at[2], ko=at[3],
                      qs=st[0], ks=st[1], qos=st[2], kos=st[3])
        assert rc in (_lib.ERR_CUDA, _lib.ERR_INVALID)
        if rc == _lib.ERR_INVALID:
            assert "overlap" in _lib.last_error()
            refused += 1
            continue
        taken += 1
        rows = [[a + 4 * (t * s[0] + h * s[1]) for t in range(tokens) for h in range(n)] for a, s, n in zip(at, st, (hq, hk) * 2)]
        sets = [{r + 4 * e for r in x for e in range(d)} for x in rows]
        for i in (2, 3):
            assert len(sets[i]) == len(rows[i]) * d             # an output's own rows are apart
            for j in range(4):
                if j != i and not (j == i - 2 and rows[i] == rows[j]):
                    assert not sets[i] & sets[j], (d, tokens, hq, hk, at, st)
    assert taken > 1000 and refused > 1000


def test_write_takes_caches_of_the_largest_sizes_that_are_checked():
    """Sizes whose bytes pass 64 bits are of no memory; the checks come to an end on them."""
    keep, at = _cache(pages=(1 << 31) - 1, page=(1 << 31) - 1, heads_=65536)
    assert L.rmsnorm_qk_rope_write(_rope(v=V, slots=SLOTS, cache=at, ko=0, hk=65536, tokens=1), None) in \
        (_lib.ERR_CUDA, _lib.ERR_INVALID)
