"""The check that bench.py's attention mode runs after its timed region, on the CPU: it passes
for outputs made from the formulas and counts planted mistakes."""
import sys

import pytest
import torch

import heads_oracle as H
from conftest import ROOT

sys.path.insert(0, ROOT)
import bench  # noqa: E402
import rmsnorm_tp_b200 as rtp  # noqa: E402

E4M3 = torch.float8_e4m3fn


class _Cache:
    """What the check asks of a cache, over rows by slot."""

    def __init__(self, k, v, page_size, dtype):
        self.rows, self.page_size, self.dtype = [k, v], page_size, dtype

    def read(self, slots, dtype):
        return tuple(r[slots].to(dtype) for r in self.rows)


def _step(held):
    """A decode step of five sequences: the check's arguments."""
    batch, hq, hk, d, page, eps = 5, 4, 2, 64, 16, 1e-6
    g = torch.Generator().manual_seed(3)
    normal = lambda *n: torch.randn(*n, generator=g)  # noqa: E731
    q, k, v = (normal(batch, h, d).bfloat16() for h in (hq, hk, hk))
    w, rope = (1 + 0.1 * normal(d)).bfloat16(), rtp.rope_table(128, d)
    lens = torch.tensor([70, 1, 33, 64, 17])
    table = torch.randperm(25, generator=g).view(batch, 5).to(torch.int32)
    pos = lens - 1
    slots = table.gather(1, (pos // page)[:, None])[:, 0].long() * page + pos % page

    def kept(x):
        """As the cache holds it."""
        if held != E4M3:
            return x.to(held).double()
        scale = x.abs().amax(-1, keepdim=True) / 448
        return (x / scale).float().to(E4M3).double() * scale

    cache = _Cache(kept(normal(25 * page, hk, d).double()), kept(normal(25 * page, hk, d).double()), page, held)
    cache.rows[0][slots] = kept(H.forward(k, w, rope, pos, eps, False)[0])
    cache.rows[1][slots] = kept(v.double())
    turned = H.forward(q, w, rope, pos, eps, False)[0].bfloat16()
    out = torch.empty_like(turned)
    for b in range(batch):
        t = torch.arange(int(lens[b]))
        kk, vv = (r[table[b][t // page].long() * page + t % page].transpose(0, 1).repeat_interleave(2, 0) for r in cache.rows)
        p = torch.softmax(torch.einsum("hd,hnd->hn", turned[b].double(), kk) * d ** -0.5, -1)
        out[b] = torch.einsum("hn,hnd->hd", p, vv).bfloat16()
    return [q, k, v, w, rope, pos, cache, slots, table, lens, turned, out]


@pytest.mark.parametrize("held", [torch.bfloat16, E4M3])
def test_the_check_passes_right_outputs_and_counts_mistakes(held):
    got = bench.attention_parity(*_step(held))
    assert got["bad"] == 0 and got["sequences"] == 3 and got["worst_of_bound"] <= 1
    assert got["checked"] == 3 * (4 + 2 + 2 + 4) * 64
    for plant in ("turned", "out", "k", "v", "nan"):
        a = _step(held)
        cache, slots, turned, out = a[6], a[7], a[10], a[11]
        if plant == "turned":
            turned[2, 1, 5] += 0.25
        elif plant == "out":
            out[4, 3] = out[4, 2]
        elif plant == "nan":
            out[0, 0, 0] = float("nan")
        else:
            cache.rows["kv".index(plant)][slots[0], 1] = cache.rows["kv".index(plant)][slots[2], 1]
        assert bench.attention_parity(*a)["bad"] > 0, plant


def test_other_ranks_leave_before_a_gpu_is_asked_for(monkeypatch):
    monkeypatch.setenv("WORLD_SIZE", "2")
    monkeypatch.setenv("RANK", "1")
    monkeypatch.setenv("LOCAL_RANK", "1")
    assert bench.run_attention_bench(bench.parse_args(["--op", "attention"])) == 0
