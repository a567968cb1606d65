"""Operands of the operators on heads that share memory, as the C entry points judge them
(without a GPU: accepted calls end at a device that does not exist)."""
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
