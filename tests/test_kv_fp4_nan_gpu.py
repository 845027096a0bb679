"""NaN keys and values that only some of a request's rows see, in all forms of attention over the 4-bit K/V pool."""
import math

import pytest
import torch

import plain_kv_fp4 as plain
from minisglang_rdna4_b200 import ops

pytestmark = pytest.mark.gpu

PAGE = 32
# (request, token, key head, channel): the block of 16 channels around it
PLACES = [(0, 0, 0, 5), (0, 37, -1, 16), (0, 170, 0, 63), (0, 171, 0, 20), (0, 250, 0, 0), (1, 128, -1, 30), (2, 100, 0, 1), (2, 505, 0, 33),
          (2, 506, -1, 47), (2, 640, 0, 9), (3, 38, 0, 60), (4, 4, -1, 2)]


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _sees(m, n, window):
    """[rows, tokens]: what the last m positions of n see."""
    i, p = torch.arange(n), n - m + torch.arange(m)[:, None]
    return (i <= p) & (i > p - (window or n + 1))


def _check(where, hq, hk, dim, dtype, window, form, news=(300, 128, 200, 3, 1)):
    lens = [300, 129, 700, 40, 5]
    width, need = 22, [-(-n // PAGE) for n in lens]
    g = torch.Generator("cuda").manual_seed(dim + hq)
    order = torch.randperm(sum(need) + 1, generator=g, device="cuda").tolist()
    table = torch.full((len(lens), width), order[-1], dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n], order = torch.tensor(order[:n], dtype=torch.int32), order[n:]
    pages = sum(need) + 1
    cache = torch.zeros(pages, hk, PAGE // 16, 18 * dim, dtype=torch.uint8, device="cuda")
    k, v = (torch.randn(pages * PAGE, hk, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    for b, t, h, c in PLACES:
        (k if where == "key" else v)[int(table[b, t // PAGE]) * PAGE + t % PAGE, h % hk, c] = math.nan
    ks, vs = (0.02 + 0.01 * torch.rand(hk, generator=g, device="cuda") for _ in range(2))
    ops.store_kv_fp4(k, v, cache, torch.arange(pages * PAGE, dtype=torch.int32, device="cuda"), ks, vs)
    table = table.cuda()
    cu = _ints([0] + torch.tensor(news).cumsum(0).tolist())
    q = torch.randn(sum(news), hq, dim, generator=g, device="cuda").to(dtype)
    weights = torch.rand(pages, hk, PAGE, generator=g, device="cuda") if form == "weights" else None
    before = weights.clone() if weights is not None else None
    p = None
    if form == "plan":
        p = ops.prefill_plan_fp4(q, cache, cu.cpu().numpy(), _ints(lens).cpu().numpy(), window)
        assert p is not None
    out = ops.paged_attention_fp4(q, cache, table, cu, _ints(lens), 0.1, k_scale=ks, v_scale=vs, window=window, max_q=max(news),
                                  plan=p, weights=weights).cpu()
    values = plain.values(cache, ks, vs)
    want, tol, w, w_tol = plain.attention(q, *values, table, cu, _ints(lens), 0.1, window)
    if form == "plan" and dtype == torch.bfloat16:
        # probabilities of 8 bits in place of 11: 2^-8 of the sum of weighted magnitudes more, the attention over the magnitudes
        tol = tol + 2.0 ** -8 * plain.attention(q, values[0], values[1].nan_to_num().abs(), table, cu, _ints(lens), 0.1, window)[0]
    bad = torch.zeros(out.shape, dtype=torch.bool)
    given = [torch.zeros(hk, n, dtype=torch.bool) for n in lens]
    group = hq // hk
    for b, t, h, c in PLACES:
        h, rows = h % hk, slice(int(cu[b]), int(cu[b + 1]))
        sees = _sees(news[b], lens[b], window)
        if where == "key":
            bad[rows, h * group:(h + 1) * group] |= sees[:, t][:, None, None]
            given[b][h] |= sees[sees[:, t]].any(0)
        else:
            bad[rows, h * group:(h + 1) * group, c // 16 * 16:c // 16 * 16 + 16] |= sees[:, t][:, None, None]
    assert bad.any() and not bad.all()
    assert torch.equal(out.isnan(), bad)
    off = (out.double() - want).abs()
    assert (off <= tol)[~bad].all(), float((off / tol)[~bad].max())
    if weights is None:
        return
    expect, room = before.cpu().double(), torch.zeros(before.shape, dtype=torch.float64)
    none = torch.zeros(before.shape, dtype=torch.bool)
    for b, n in enumerate(lens):
        i = torch.arange(n)
        at = (table[b].cpu().long()[i // PAGE], slice(None), i % PAGE)
        expect[at] += w[b].T
        room[at] += w_tol[b].T
        none[at] = given[b].T
    room = room + expect * 2.0 ** -22                       # sums over the heads and with what was there
    weights = weights.cpu()
    assert torch.equal(weights.isnan(), none)
    assert ((weights.double() - expect).abs() <= room)[~none].all()


SHAPES = [(8, 2, 128), (7, 1, 64), (8, 4, 64), (16, 1, 128)]


@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("window", [0, 70, 300])
@pytest.mark.parametrize("hq,hk,dim", SHAPES)
def test_rows_of_the_general_form(where, window, hq, hk, dim):
    _check(where, hq, hk, dim, torch.bfloat16, window, "")
    _check(where, hq, hk, dim, torch.float16, window, "weights")


@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("window", [0, 20])
def test_wide_heads_and_few_rows(where, window):
    _check(where, 8, 2, 256, torch.bfloat16, window, "weights")
    _check(where, 4, 2, 128, torch.bfloat16, window, "weights", (4, 4, 4, 3, 1))       # no more than 8 rows a key head


@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("window", [0, 70, 300])
@pytest.mark.parametrize("hq,hk,dim", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_prompts(where, window, hq, hk, dim, dtype):
    _check(where, hq, hk, dim, dtype, window, "plan")
