"""GPU: attention over pages whose value scales lie far apart, against the formula in 64 bits.

Tolerance of an output, with l = sum exp(s - max), p the weights, v = 2^lv c, and TOP the largest value exponent of the sequence's pages:
  2^-8 |o|                                   the result's rounding to bf16
  (2^-11 + 3 delta) sum p |v|                a weight's rounding to f16, and what the query's rounding moves it (as in test_gpu_kv8.py)
  sum |c| 2^-25 max(2^(lv + 8), 2^(TOP - 70)) / l   weights below the normal range of f16: the unit of the outputs is 2^(R - 8) at most, R at most
                                             lv + 8 (16 are allowed here; the last test is closer), or TOP + 2 - 64 where it may not follow
  2^(TOP - 142) / l                          what was summed before the unit rose to 2^(TOP + 2 - 8), below f32's smallest number"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cache(cuda, exps, ps, d, seed, zero=(), kvh=2):
    """One sequence that fills pages of the given value exponents, in a shuffled pool; the pages of `zero` hold codes of 0."""
    from oxicuda_b200.kv_cache import PagedFp8KvCache
    g = torch.Generator(device=cuda).manual_seed(seed)
    n = len(exps)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).to(cuda)
    codes = [(100 * torch.randn(n, kvh, ps, d, device=cuda, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2)]
    v_scales = torch.zeros(n, kvh, dtype=torch.uint8, device=cuda)
    v_scales[order] = (torch.tensor(exps, device=cuda) + 127).to(torch.uint8)[:, None].expand(n, kvh)
    for i in zero:
        codes[1][order[i]] = 0
    cache = PagedFp8KvCache(codes[0], codes[1], torch.full((n, kvh), 120, dtype=torch.uint8, device=cuda), v_scales)
    return cache, order.to(torch.int32)[None].contiguous()


def _check(cache, table, exps, n, new, q, out):
    d, ps, kvh = cache.head_dim, cache.page_size, cache.n_kv_heads
    group, scale, top_exp = q.shape[1] // kvh, d ** -0.5, max(exps)
    pages = table[0].long()
    lv = (cache.v_scales[pages, 0].double() - 127).repeat_interleave(ps)[:n]
    see = torch.arange(n, device=q.device)[None] <= (n - new + torch.arange(new, device=q.device))[:, None]
    for h in range(kvh):
        k = (cache.k_codes[pages, h].view(torch.float8_e4m3fn).double() * 2.0 ** -7).reshape(-1, d)[:n]
        c = cache.v_codes[pages, h].view(torch.float8_e4m3fn).double().reshape(-1, d)[:n]
        v = c * torch.exp2(lv)[:, None]
        qq = q[:, h * group: (h + 1) * group].double()
        s = (torch.einsum("qgd,kd->gqk", qq, k) * scale).masked_fill(~see[None], -math.inf)
        e = torch.exp(s - s.amax(dim=2, keepdim=True))
        l = e.sum(dim=2, keepdim=True)
        ref, A = torch.einsum("gqk,kd->qgd", e / l, v), torch.einsum("gqk,kd->qgd", e / l, v.abs())
        low = c.abs() * 2.0 ** -25 * torch.exp2(torch.clamp(lv + 8, min=top_exp - 70))[:, None]
        floor = torch.einsum("gqk,kd->qgd", see[None].double().expand_as(e) / l, low) + 2.0 ** (top_exp - 142) / l.permute(1, 0, 2)
        delta = scale * qq.abs().amax(dim=2) * (k.abs().sum(dim=1)[None] * see).amax(dim=1)[:, None] * (2.0 ** -17 + 2.0 ** -16)
        got = out[:, h * group: (h + 1) * group].double()
        tol = 2.0 ** -8 * ref.abs() + (2.0 ** -11 + 3 * delta[..., None]) * A + floor
        bad = ~((got - ref).abs() <= tol)
        assert not bad.any(), (h, int(bad.sum()), got[bad][0].item(), ref[bad][0].item(), tol[bad][0].item())


def _run(cuda, exps, ps, d, new, seed, zero=(), group=4):
    from oxicuda_b200 import _lib as L
    cache, table = _cache(cuda, exps, ps, d, seed, zero)
    n = len(exps) * ps - 3
    g = torch.Generator(device=cuda).manual_seed(seed + 1)
    q = (0.7 * torch.randn(new, 2 * group, d, device=cuda, generator=g)).to(torch.bfloat16)
    starts = None if new == 1 else torch.tensor([0, new], dtype=torch.int32, device=cuda)
    out = cache.attend(q, torch.tensor([n], dtype=torch.int32, device=cuda), table, q_starts=starts)
    L.default_handle().check()
    _check(cache, table, exps, n, new, q, out)


@pytest.mark.parametrize("ps,d", [(16, 128), (64, 128), (128, 64)])
@pytest.mark.parametrize("new", [1, 3, 60])
@pytest.mark.parametrize("big", [20, 58, 90, 119])
def test_zero_pages_behind_large_ones(cuda, ps, d, new, big):
    """A page of zeros has the smallest scale there is: outputs summed in the unit of pages of 2^20 to 2^119 stay finite and right."""
    pages = max(12, 512 // ps)
    exps = [big] * pages + [-50] * pages
    _run(cuda, exps, ps, d, new, big + ps, zero=range(pages, 2 * pages))
    _run(cuda, [big if i % 3 == 0 else -50 for i in range(2 * pages)], ps, d, new, big, zero=[i for i in range(2 * pages) if i % 3])


@pytest.mark.parametrize("ps,d", [(16, 64), (64, 128)])
@pytest.mark.parametrize("new", [1, 4, 40])
@pytest.mark.parametrize("gap", [9, 30, 60])
def test_small_values_behind_large_scales(cuda, ps, d, new, gap):
    """Pages of a large scale whose codes are 0: the rest, up to 2^60 smaller, is all there is, and keeps its precision."""
    pages = max(12, 512 // ps)
    _run(cuda, [40] * pages + [40 - gap] * pages, ps, d, new, gap + ps, zero=range(pages))


@pytest.mark.parametrize("ps,d", [(16, 128), (64, 64)])
@pytest.mark.parametrize("new", [2, 4, 200])
@pytest.mark.parametrize("low,high", [(-30, 110), (-45, 85), (0, 60)])
def test_rows_that_do_not_see_the_large_pages_behind_them(cuda, ps, d, new, low, high):
    """The last rows see a page of far larger values: what the rows in front of it have summed is brought to its unit, and comes out the same."""
    pages = max(4, 512 // ps)
    _run(cuda, [low] * (pages - 1) + [high], ps, d, new, low + high + ps, group=1 if new == 2 else 4)
    _run(cuda, [low] * (pages - 1) + [high] * 3, ps, d, min(new, 3 * ps), high + ps)


@pytest.mark.parametrize("new,top,lead,low,score", [(1, 8, 0, -8, 13.5958), (32, 16, 10, 2, 8.7437)])
def test_small_weights_on_pages_of_a_smaller_scale(cuda, new, top, lead, low, score):
    """Many keys of one small weight on the smallest of pages that are multiplied together: e^-13.6 and e^-8.7 lie 0.45 steps above a number of f16's
    subnormal range if they enter as p * 2^-1 and p * 2^-8, 4 % off.  All of the output comes from them."""
    from oxicuda_b200.kv_cache import PagedFp8KvCache
    ps, d, front, pairs = 16, 128, 96, 48
    exps = [top] * front + [lead, low] * pairs
    g = torch.Generator(device=cuda).manual_seed(new)
    n = len(exps)
    k = torch.zeros(n, 1, ps, d, dtype=torch.uint8, device=cuda)
    k[front:, :, :, 0] = 0xB8                              # -1: these keys score -score, those in front 0
    v = (100 + 50 * torch.rand(n, 1, ps, d, device=cuda, generator=g)).to(torch.float8_e4m3fn).view(torch.uint8)
    v[:front] = 0
    v[front::2] = 0
    scales = (torch.tensor(exps, device=cuda) + 127).to(torch.uint8)[:, None].contiguous()
    cache = PagedFp8KvCache(k, v, torch.full_like(scales, 127), scales)
    q = torch.zeros(new, 4, d, dtype=torch.bfloat16, device=cuda)
    q[..., 0] = 1
    keys = n * ps
    starts = None if new == 1 else torch.tensor([0, new], dtype=torch.int32, device=cuda)
    out = cache.attend(q, torch.tensor([keys], dtype=torch.int32, device=cuda), torch.arange(n, dtype=torch.int32, device=cuda)[None].contiguous(), q_starts=starts,
                       scale=score)
    value = (v.view(torch.float8_e4m3fn).double() * torch.exp2(torch.tensor(exps, device=cuda).double())[:, None, None, None]).view(keys, d)
    s = torch.where(torch.arange(keys, device=cuda) < front * ps, 0.0, -score).double()
    see = torch.arange(keys, device=cuda)[None] <= (keys - new + torch.arange(new, device=cuda))[:, None]
    p = torch.exp(s)[None] * see
    want = ((p @ value) / p.sum(dim=1, keepdim=True))[:, None].expand(new, 4, d)
    # 2^-8 the result, 2^-11 a weight, 2^-25 of the largest weight (1) against a weight of e^-score, 2^-19 the exponentials and sums in f32
    tol = 2.0 ** -8 + 2.0 ** -11 + 2.0 ** -25 * math.exp(score) + 2.0 ** -19
    assert ((out.double() - want).abs() <= tol * want.abs()).all(), ((out.double() - want).abs() / want).max()


def test_rows_beside_a_bad_page_are_right(cuda):
    """A table entry that names no page is left out of its own sequence, with and without row offsets; the others come out as they should."""
    from oxicuda_b200 import _lib as L
    from tests.test_gpu_kv8 import _check as check, _pages, _q
    for new in (1, 3, 40):
        lens = [40, 50, 60, 70]
        cache, table = _pages(cuda, lens, 16, 2, 128, 14)
        q = _q(cuda, 4 * new, 8, 128, 3)
        seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
        bad = table.clone()
        bad[0, 1], bad[3, 0] = cache.num_pages, -5
        for starts in ((None,) if new == 1 else ()) + (torch.arange(0, 4 * new + 1, new, dtype=torch.int32, device=cuda),):
            out = cache.attend(q, seq, bad, q_starts=starts)
            with pytest.raises(L.InvalidArgument):
                L.default_handle().check()
            assert torch.isfinite(out).all()
            check(cache, table[1:3], lens[1:3], [new, new], q[new: 3 * new], out[new: 3 * new])
            # the keys of the pages that are there, by definition
            pos = lens[0] - new + torch.arange(new, device=cuda)
            j = torch.tensor([i for i in range(lens[0]) if i // 16 != 1], device=cuda)
            for h in range(2):
                pages = table[0, j // 16].long()
                k, v = [c[pages, h, j % 16].view(torch.float8_e4m3fn).double() * torch.exp2(s[pages, h].double() - 127)[:, None]
                        for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales))]
                qq = q[:new, 4 * h: 4 * h + 4].double()
                s = (torch.einsum("qgd,kd->gqk", qq, k) * 128 ** -0.5).masked_fill(~(j[None] <= pos[:, None])[None], float("-inf"))
                p = torch.softmax(s, dim=2)
                want, A = torch.einsum("gqk,kd->qgd", p, v), torch.einsum("gqk,kd->qgd", p, v.abs())
                delta = 128 ** -0.5 * qq.abs().amax(dim=2) * k.abs().sum(dim=1).amax() * (2.0 ** -17 + 2.0 ** -16)
                err = (out[:new, 4 * h: 4 * h + 4].double() - want).abs()
                assert (err <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 3 * delta[..., None]) * A + 2.0 ** -17 * v.abs().sum(dim=0)).all()
