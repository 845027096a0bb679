"""Eviction from the 4-bit K/V pool: calls whose bounds or pages are not what the step has."""
import pytest
import torch

from minisglang_rdna4_b200 import ops
from minisglang_rdna4_b200.ops import ref_fp4

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _case(lens, budget, hk=2, page=16, dim=64, layers=2, seed=0):
    """``(cache, weights, table, lengths, new table)``: pages of the requests and new ones, and two that belong to nobody (the first and
    the last)."""
    need = [-(-n // page) for n in lens]
    slim, pages = -(-budget // page), sum(need) + len(lens) * -(-budget // page) + 2
    g = torch.Generator("cuda").manual_seed(seed)
    cache = torch.randint(0, 256, (layers, pages, hk, page // 16, 18 * dim), generator=g, device="cuda", dtype=torch.uint8)
    weights = torch.round(torch.rand(layers, pages, hk, page, generator=g, device="cuda") ** 3 * 60)
    order = (1 + torch.randperm(pages - 2, generator=torch.Generator().manual_seed(seed))).tolist()
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n], order = torch.tensor(order[:n], dtype=torch.int32), order[n:]
    return cache, weights, table.cuda(), _ints(lens), _ints(order).view(len(lens), slim)


@pytest.mark.parametrize("max_kv", [1, 40, 255, 256, 1 << 33])
@pytest.mark.parametrize("lens,budget,recent,sinks", [([300, 20, 77, 1000], 33, 6, 3), ([50021, 90], 1025, 3, 13)])
def test_requests_longer_than_said_lose_nothing(lens, budget, recent, sinks, max_kv):
    cache, weights, table, n, new = _case(lens, budget)
    want, want_w = cache.clone(), weights.clone()
    stay, now = ref_fp4.evict_kv_fp4(want, want_w, table, n, new, budget, recent, sinks)
    kept, got_now = ops.evict_kv_fp4(cache, weights, table, n, new, budget, recent, sinks, max_kv=max_kv)
    assert torch.equal(got_now, now.to(got_now)) and torch.equal(kept, stay)
    assert torch.equal(cache, want) and torch.equal(weights, want_w)


def test_new_pages_outside_the_pool_are_written_nowhere():
    """Pages below 0 and behind the pool in the new table: the pool's first and last page stay as they are, the other new pages get
    their rows, and what is kept is as ever."""
    lens, budget = [300, 20, 77, 500], 40
    cache, weights, table, n, new = _case(lens, budget)
    pages = cache.shape[1]
    whole, whole_w = cache.clone(), weights.clone()
    stay, now = ref_fp4.evict_kv_fp4(whole, whole_w, table, n, new, budget, 6, 3)
    bad = new.clone()
    bad[0, 1], bad[1, 0], bad[2, 2], bad[3] = -1, pages, 1 << 30, -(1 << 31)
    want, want_w = cache.clone(), weights.clone()
    good = new[bad == new].long()
    want[:, good], want_w[:, good] = whole[:, good], whole_w[:, good]
    kept, got_now = ops.evict_kv_fp4(cache, weights, table, n, bad, budget, 6, 3)
    assert torch.equal(got_now, now.to(got_now)) and torch.equal(kept, stay)
    assert torch.equal(cache, want) and torch.equal(weights, want_w)
