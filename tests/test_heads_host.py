"""The operators on heads without a GPU: argument checks of the C entry points (they run
before any CUDA call), structure sizes, the Python surface's checks, and the oracle
itself against finite differences."""
import ctypes
import os
import subprocess

import pytest
import torch

import heads_oracle as H
import rmsnorm_tp_b200 as rtp
from conftest import ROOT
from rmsnorm_tp_b200 import _lib, heads

L = _lib.LIB
# addresses that a refused call never follows; device -1 makes an accepted one end in
# cudaSetDevice, before any launch
Q, K, V, QO, KO, W, TABLE, POS, SLOTS = (0x10000000 * i for i in range(1, 10))


def _cache(pages=4, page=16, heads_=2, dim=64, dtype=_lib.BF16, k=0xD0000000, v=0xE0000000, ks=0, vs=0):
    buf = ctypes.create_string_buffer(heads._CACHE.pack(k, v, ks, vs, pages, page, heads_, dim, dtype))
    return buf, ctypes.addressof(buf)


def _rope(q=Q, k=K, v=0, qo=QO, ko=KO, qw=W, kw=W, table=TABLE, pos=POS, qs=None, ks=None, vs=None, qos=None,
          kos=None, tokens=8, most=100, cache=0, slots=0, hq=4, hk=2, d=64, r=64, dtype=_lib.BF16, inter=0):
    n = lambda s, h: s or (h * d, d)  # noqa: E731
    return heads._ROPE_ARGS.pack(q, k, v, qo, ko, qw, kw, table, pos, *n(qs, hq), *n(ks, hk), *n(vs, hk),
                                 *n(qos, hq), *n(kos, hk), tokens, most, cache, slots, hq, hk, d, r, dtype,
                                 inter, 1e-6, -1)


def _forward(**kw):
    return L.rmsnorm_qk_rope_forward(_rope(**kw), None)


def test_structure_sizes_match_the_header(tmp_path):
    src, exe = tmp_path / "s.c", tmp_path / "s"
    src.write_text('#include "rmsnorm_tp_b200.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu %zu %zu", '
                   "sizeof(rmsnorm_qk_rope_args), sizeof(rmsnorm_qk_rope_backward_args), "
                   "sizeof(rmsnorm_kv_cache), sizeof(rmsnorm_paged_attention_args)); return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    sizes = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [s.size for s in (heads._ROPE_ARGS, heads._BACK_ARGS, heads._CACHE, heads._ATTN_ARGS)]


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(dtype=-1), dict(hq=0), dict(hk=0), dict(d=0, r=0), dict(d=514, r=64), dict(r=63), dict(r=66),
    dict(r=0), dict(most=0), dict(tokens=-1), dict(tokens=1 << 31), dict(qw=0), dict(kw=0), dict(q=0), dict(k=0),
    dict(qo=0), dict(ko=0), dict(table=0), dict(pos=0), dict(qs=(-256, 64)), dict(ks=(128, -64)),
    dict(qos=(0, 64)), dict(qos=(200, 64)), dict(kos=(128, 32)),
    dict(qo=Q + 2), dict(qo=Q, qos=(512, 64)), dict(qo=K), dict(ko=Q), dict(qo=QO, ko=QO + 512)])
def test_forward_refuses(kw):
    assert _forward(**kw) == _lib.ERR_INVALID
    assert _lib.last_error().startswith("qk_rope_forward:")


@pytest.mark.parametrize("kw", [
    dict(), dict(qw=0, kw=0), dict(qo=Q), dict(qo=Q, ko=K), dict(qs=(0, 64)), dict(qs=(256, 0)), dict(r=32, inter=1),
    # column blocks of one matrix of 8 heads a token, written where they were read
    dict(q=Q, k=Q + 512, qo=Q, ko=Q + 512, qs=(512, 64), ks=(512, 64), qos=(512, 64), kos=(512, 64)),
    dict(tokens=1, qos=(0, 64)), dict(hk=1, kos=(64, 0))])
def test_forward_takes(kw):
    assert _forward(**kw) == _lib.ERR_CUDA          # past the checks, to a device that does not exist


def test_null_arguments_and_empty_calls():
    assert L.rmsnorm_qk_rope_forward(None, None) == _lib.ERR_INVALID
    assert L.rmsnorm_qk_rope_write(None, None) == _lib.ERR_INVALID
    assert L.rmsnorm_qk_rope_backward(None, None) == _lib.ERR_INVALID
    assert L.rmsnorm_paged_attention(None, None) == _lib.ERR_INVALID
    assert L.rmsnorm_kv_read(None, None, None, None, 1, 0, 0, None) == _lib.ERR_INVALID
    assert _forward(tokens=0, q=0, k=0, qo=0, ko=0, pos=0) == _lib.OK
    ws = L.rmsnorm_qk_rope_backward_workspace_bytes
    assert ws(8192, 32, 8, 128, 128, _lib.BF16) == 1024 * 128 * 4
    assert ws(8, 4, 2, 50, 20, _lib.BF16) == 1024 * 50 * 4          # no vector rows: two kernels
    assert ws(8, 4, 2, 64, 64, _lib.BF16) == ws(0, 4, 2, 64, 64, _lib.BF16) == 0       # one cluster
    assert ws(8, 4, 2, 0, 64, _lib.BF16) == ws(-1, 4, 2, 64, 64, _lib.BF16) == ws(8, 4, 2, 64, 64, 7) == 0


@pytest.mark.parametrize("cache", [
    dict(heads_=1), dict(dim=128), dict(dtype=_lib.F16), dict(dtype=4), dict(dtype=_lib.KV_E4M3), dict(page=0),
    dict(pages=-1), dict(k=0), dict(k=0xD0000008)])
def test_write_refuses_caches(cache):
    keep, at = _cache(**cache)
    assert L.rmsnorm_qk_rope_write(_rope(v=V, slots=SLOTS, cache=at), None) == _lib.ERR_INVALID
    assert _lib.last_error().startswith("qk_rope_write:")


def test_write_checks():
    keep, at = _cache()
    call = lambda **kw: L.rmsnorm_qk_rope_write(_rope(**{**dict(v=V, slots=SLOTS, cache=at, ko=0), **kw}), None)  # noqa: E731
    assert call() == _lib.ERR_CUDA
    assert call(v=0) == call(slots=0) == call(cache=0) == call(qo=V) == _lib.ERR_INVALID
    keep2, e4m3 = _cache(dtype=_lib.KV_E4M3, ks=64, vs=64)
    assert call(cache=e4m3) == _lib.ERR_CUDA
    assert call(cache=e4m3, dtype=_lib.F32) == _lib.ERR_CUDA


def _back(dqo=Q, dko=K, q=0xB0000000, k=0xC0000000, dq=QO, dk=KO, dw=W, dkw=W, qw=W, kw=W, ws=V, nbytes=1024 * 64 * 4,
          tokens=8000, r=64):
    s = (256, 64, 128, 64)
    return L.rmsnorm_qk_rope_backward(heads._BACK_ARGS.pack(
        dqo, dko, q, k, dq, dk, dw, dkw, qw, kw, TABLE, POS, ws, nbytes, *s, *s, tokens, 100, 4, 2, 64, r, _lib.BF16, 0,
        1e-6, -1), None)


def test_backward_checks():
    assert _back() == _lib.ERR_CUDA
    assert _back(q=0, k=0, dw=0, qw=0, kw=0, ws=0, nbytes=0) == _lib.ERR_CUDA      # rotation alone
    assert _back(tokens=8, ws=0, nbytes=0) == _lib.ERR_CUDA                        # one cluster
    for kw in (dict(dw=0), dict(dkw=0), dict(ws=0), dict(nbytes=1024 * 64 * 4 - 1), dict(qw=0), dict(q=0), dict(dq=Q),
               dict(dk=0xC0000000), dict(dk=QO + 512), dict(tokens=8, dw=0), dict(tokens=8, dq=Q), dict(dqo=0), dict(r=1), dict(tokens=-1)):
        assert _back(**kw) == _lib.ERR_INVALID, kw


def _attn(cache, q=Q, out=QO, table=TABLE, lens=POS, ws=V, nbytes=1 << 30, qs=(256, 64), batch=3, pages=4, hq=4,
          dtype=_lib.BF16):
    return heads._attention_args(q, out, 0, table, lens, ws, nbytes, cache, qs, pages, batch, pages, hq, dtype, 0.1,
                                 0)


def test_attention_refuses_before_any_cuda_call():
    keep, at = _cache()
    for kw in (dict(hq=3), dict(hq=0), dict(dtype=_lib.F16), dict(dtype=9), dict(batch=-1), dict(batch=65536),
               dict(pages=-1), dict(pages=1 << 27), dict(pages=1 << 60), dict(q=0), dict(out=0), dict(lens=0), dict(table=0),
               dict(out=Q), dict(qs=(-256, 64)), dict(out=QO + 8), dict(ws=V + 4),
               dict(batch=65535, hq=65536, pages=1 << 26)):
        assert L.rmsnorm_paged_attention(_attn(at, **kw), None) == _lib.ERR_INVALID, kw
        assert _lib.last_error().startswith("paged_attention:")
    assert L.rmsnorm_paged_attention(_attn(at, batch=0, q=0, out=0), None) == _lib.OK
    keep2, odd = _cache(dim=72)
    assert L.rmsnorm_paged_attention(_attn(odd), None) == _lib.ERR_INVALID


def test_read_refuses_before_any_cuda_call():
    keep, at = _cache()
    read = lambda k=Q, v=K, slots=SLOTS, n=4, dtype=1: L.rmsnorm_kv_read(at, k, v, slots, n, dtype, -1, None)  # noqa: E731
    assert read() == _lib.ERR_CUDA and read(n=0, k=0) == _lib.OK
    assert read(k=0) == read(slots=0) == read(n=-1) == read(n=1 << 31) == read(n=1 << 62) == read(dtype=3) == read(k=Q + 2) == \
        _lib.ERR_INVALID


def test_python_surface_refuses_host_tensors_and_bad_tables():
    q, k, w = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64), torch.ones(64)
    table, pos = rtp.rope_table(16, 64), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(AssertionError, match="CUDA"):
        rtp.qk_norm_rope(q, k, w, w, table, pos)
    with pytest.raises(AssertionError, match="CUDA"):
        rtp.PagedKVCache.from_tensors(torch.zeros(1, 1, 16, 64), torch.zeros(1, 1, 16, 64))
    for bad in ((0, 64), (16, 63), (16, 0)):
        with pytest.raises(AssertionError):
            rtp.rope_table(*bad)


def test_rope_table_is_right_at_far_positions():
    table = rtp.rope_table(100001, 8, base=500000.0)
    assert table.shape == (100001, 8) and table.dtype == torch.float32
    import math
    for i in range(4):
        angle = 100000 * 500000.0 ** (-2 * i / 8)
        assert abs(table[100000, i].item() - math.cos(angle)) < 1e-7
        assert abs(table[100000, 4 + i].item() - math.sin(angle)) < 1e-7


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_gradients_against_differences(interleaved):
    """The oracle's backward against central differences of its forward: h = 1e-5 leaves
    an error of h^2 (third derivatives, of the order of one) and 2^-52 / h."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 2, 10, generator=g, dtype=torch.float64)
    w = 1 + 0.1 * torch.randn(10, generator=g, dtype=torch.float64)
    dy = torch.randn(3, 2, 10, generator=g, dtype=torch.float64)
    rope, pos = rtp.rope_table(50, 6), torch.tensor([0, 7, 49])
    dx, _, dw, _ = H.backward(dy, x, w, rope, pos, 1e-3, interleaved)
    loss = lambda x, w: (H.forward(x, w, rope, pos, 1e-3, interleaved)[0] * dy).sum().item()  # noqa: E731
    h = 1e-5
    for t, grad in ((x, dx), (w, dw)):
        flat = t.view(-1)
        for i in range(0, flat.numel(), 7):
            keep = flat[i].item()
            flat[i] = keep + h
            up = loss(x, w)
            flat[i] = keep - h
            down = loss(x, w)
            flat[i] = keep
            assert abs((up - down) / (2 * h) - grad.reshape(-1)[i].item()) < 1e-7
