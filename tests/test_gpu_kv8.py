"""GPU: the paged E4M3 cache (append) and the attention that reads it, against plain statements in 64 bits.

Tolerance of an output.  bf16 rounds by 2^-8 of the value.  A query element is off by at most 2^-17 of its row's largest, so a score by
d = 2^-17 max|q| sum_c |k_c| * scale plus f32 sums (128 additions of at most 2^-23 of sum |q k|); that moves the weights by e^(2 d) - 1 <= 3 d of
themselves.  A weight is off by 2^-9 of itself, or by 2^-18 of the row's largest (2^-14 where the value scales of pages differ by up to
2^4) below the normal range.  With A = sum p |v| and B = sum |v| / sum exp(s - max):
  |err| <= 2^-8 |o| + (2^-8 + 3 d) A + 2^-13 B * 2^-1."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _pages(cuda, lens, ps, kvh, d, seed, spread=0.3, extra=3, jump=0):
    """A random cache for sequences of the given lengths; stale slots and unused pages hold NaN codes and scale bytes of 255."""
    from oxicuda_b200.kv_cache import PagedFp8KvCache
    g = torch.Generator(device=cuda).manual_seed(seed)
    pages = [-(-n // ps) for n in lens]
    num = sum(pages) + extra
    order = torch.randperm(num, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(1, max(pages)) + 1
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    used, at = torch.zeros(num, dtype=torch.bool), 0
    for b, p in enumerate(pages):
        table[b, :p] = torch.tensor(order[at: at + p], dtype=torch.int32)
        used[order[at: at + p]] = True
        at += p
    out = []
    for _ in range(2):
        x = torch.randn(num, kvh, ps, d, device=cuda, generator=g).clamp(-3.4, 3.4) * 100
        codes = x.to(torch.float8_e4m3fn).view(torch.uint8)
        scales = (127 - 7 + (spread * torch.randn(num, kvh, device=cuda, generator=g)).round() +
                  (jump * torch.randint(0, 2, (num, kvh), device=cuda, generator=g) if jump else 0)).to(torch.uint8)
        scales[~used.to(cuda)] = 255
        codes[~used.to(cuda)] = 0x7F
        for b, n in enumerate(lens):
            if n % ps:
                codes[table[b, n // ps].item(), :, n % ps:] = 0x7F
        out.append((codes, scales))
    cache = PagedFp8KvCache(out[0][0], out[1][0], out[0][1], out[1][1])
    return cache, table.to(cuda)


def _dense(codes, scales, pages, n, h):
    """[n, d] in 64 bits: the first n tokens of head h."""
    v = codes[pages, h].view(torch.float8_e4m3fn).double() * torch.exp2(scales[pages, h].double() - 127)[:, None, None]
    return v.reshape(-1, v.shape[-1])[:n]


def _check(cache, table, lens, news, q, out, lse=None, scale=None, window=0, r0s=None):
    d = cache.head_dim
    scale = d ** -0.5 if scale is None else scale
    group = q.shape[1] // cache.n_kv_heads
    r0 = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        if r0s is not None:
            r0 = r0s[b]
        if m == 0:
            continue
        pages = table[b, : -(-n // cache.page_size)].long()
        pos = n - m + torch.arange(m, device=q.device)
        j = torch.arange(n, device=q.device)
        see = j[None] <= pos[:, None]
        if window:
            see &= j[None] > pos[:, None] - window
        for h in range(cache.n_kv_heads):
            k, v = _dense(cache.k_codes, cache.k_scales, pages, n, h), _dense(cache.v_codes, cache.v_scales, pages, n, h)
            qq = q[r0: r0 + m, h * group: (h + 1) * group].double()
            s = torch.einsum("qgd,kd->gqk", qq, k) * scale
            s = s.masked_fill(~see[None], -math.inf)
            top = s.amax(dim=2, keepdim=True)
            e = torch.exp(s - top)
            l = e.sum(dim=2, keepdim=True)
            ref = torch.einsum("gqk,kd->qgd", e / l, v)
            A = torch.einsum("gqk,kd->qgd", e / l, v.abs())
            B = torch.einsum("gqk,kd->qgd", see[None].double().expand_as(e) / l, v.abs())
            qmax = qq.abs().amax(dim=2)                                            # [q, g]
            ksum = (k.abs().sum(dim=1)[None] * see).amax(dim=1)                    # [q]
            delta = abs(scale) * qmax * ksum[:, None] * (2.0 ** -17 + 2.0 ** -16)   # the second term: 128 * 2^-23
            got = out[r0: r0 + m, h * group: (h + 1) * group].double()
            tol = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 3 * delta[..., None]) * A + 2.0 ** -14 * B
            bad = (got - ref).abs() > tol
            assert not bad.any() and torch.isfinite(got).all(), (b, h, int(bad.sum()), float(((got - ref).abs() / tol).max()))
            if lse is not None:
                want = (top + torch.log(l))[..., 0].t()
                assert ((lse[r0: r0 + m, h * group: (h + 1) * group].double() - want).abs() <= delta + 1e-5 + 1e-6 * want.abs()).all()
        r0 += m


def _starts(news, cuda):
    s = [0]
    for n in news:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device=cuda)


def _q(cuda, rows, heads, d, seed, size=1.3):
    g = torch.Generator(device=cuda).manual_seed(seed + 77)
    return (size * torch.randn(rows, heads, d, device=cuda, generator=g)).to(torch.bfloat16)


# ---- attention --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("kvh,group", [(1, 1), (2, 4), (1, 7), (2, 8), (1, 12), (3, 16)])
def test_decode(cuda, d, ps, kvh, group):
    lens = [1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 129, 500, 1003]
    cache, table = _pages(cuda, lens, ps, kvh, d, d + ps + group)
    q = _q(cuda, len(lens), kvh * group, d, ps)
    out, lse = cache.attend(q, torch.tensor(lens, dtype=torch.int32, device=cuda), table, want_lse=True)
    _check(cache, table, lens, [1] * len(lens), q, out, lse)


@pytest.mark.parametrize("d,ps", [(64, 16), (128, 16), (128, 64), (64, 128)])
@pytest.mark.parametrize("news,olds", [
    ([1], [0]), ([2], [0]), ([5, 0, 1], [0, 9, 300]), ([4] * 6, [0, 1, 15, 60, 127, 700]), ([17, 130], [3, 0]), ([64, 1, 33], [64, 1000, 31]),
    ([128], [128]), ([129, 255], [1, 257]), ([300], [500]), ([512, 3], [0, 1500])])
def test_ragged_prefill(cuda, d, ps, news, olds):
    lens = [n + o for n, o in zip(news, olds)]
    for kvh, group in ((2, 4), (1, 7), (2, 1)):
        cache, table = _pages(cuda, lens, ps, kvh, d, sum(lens) + d + ps)
        q = _q(cuda, sum(news), kvh * group, d, sum(news))
        out, lse = cache.attend(q, torch.tensor(lens, dtype=torch.int32, device=cuda), table, q_starts=_starts(news, cuda), want_lse=True)
        _check(cache, table, lens, news, q, out, lse)


@pytest.mark.parametrize("window", [1, 7, 32, 100, 5000])
@pytest.mark.parametrize("news,olds", [([1, 1, 1], [0, 40, 700]), ([3, 200, 70], [50, 0, 333]), ([400], [100])])
def test_window(cuda, window, news, olds):
    lens = [n + o for n, o in zip(news, olds)]
    cache, table = _pages(cuda, lens, 32, 2, 128, window)
    q = _q(cuda, sum(news), 8, 128, window)
    starts = None if max(news) == 1 else _starts(news, cuda)
    out, lse = cache.attend(q, torch.tensor(lens, dtype=torch.int32, device=cuda), table, q_starts=starts, window=window, want_lse=True)
    _check(cache, table, lens, news, q, out, lse, window=window)


@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("window", [5, 50, 100])
@pytest.mark.parametrize("new", [1, 3, 90])
def test_pages_in_front_of_the_window_may_be_gone(cuda, ps, window, new):
    """What no row's window reaches is not looked up: its owner may have given the pages back, and that is no error."""
    from oxicuda_b200 import _lib as L
    lens, news = [700, 333, 40 + new], [new] * 3
    cache, table = _pages(cuda, lens, ps, 2, 128, ps + window)
    q = _q(cuda, 3 * new, 8, 128, new)
    seq, starts = torch.tensor(lens, dtype=torch.int32, device=cuda), None if new == 1 else _starts(news, cuda)
    want = cache.attend(q, seq, table, q_starts=starts, window=window)
    gone = table.clone()
    for b, n in enumerate(lens):
        gone[b, : max(0, n - new - window + 1) // ps] = -1
    out, lse = cache.attend(q, seq, gone, q_starts=starts, window=window, want_lse=True)
    L.default_handle().check()
    assert torch.equal(out, want)
    _check(cache, table, lens, news, q, out, lse, window=window)


@pytest.mark.parametrize("ps,d", [(16, 64), (64, 128)])
def test_many_sequences(cuda, ps, d):
    """More sequences than a warp has lanes, many of them without rows."""
    g = torch.Generator().manual_seed(3)
    olds = torch.randint(0, 200, (100,), generator=g).tolist()
    for top in (3, 40):
        news = (torch.randint(0, top, (100,), generator=g) * torch.randint(0, 2, (100,), generator=g)).tolist()
        news[:33] = [0] * 33
        lens = [max(1, a + b) for a, b in zip(news, olds)]
        cache, table = _pages(cuda, lens, ps, 2, d, top)
        q = _q(cuda, sum(news), 8, d, top)
        k, v = [_q(cuda, sum(news), 2, d, i) for i in (1, 2)]
        seq, starts = torch.tensor(lens, dtype=torch.int32, device=cuda), _starts(news, cuda)
        want = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
        _append_ref(want[0], want[1], k, lens, news, table, ps)
        _append_ref(want[2], want[3], v, lens, news, table, ps)
        cache.append(k, v, seq, table, q_starts=starts)
        for w, t in zip(want, (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)):
            assert torch.equal(w, t)
        out, lse = cache.attend(q, seq, table, q_starts=starts, want_lse=True)
        _check(cache, table, lens, news, q, out, lse)


@pytest.mark.parametrize("new", [1, 2, 5])
@pytest.mark.parametrize("group", [33, 64, 128, 200])
def test_large_groups(cuda, group, new):
    lens = [90, 5, 400]
    cache, table = _pages(cuda, lens, 16, 1, 128, group)
    q = _q(cuda, 3 * new, group, 128, new)
    seq, starts = torch.tensor(lens, dtype=torch.int32, device=cuda), None if new == 1 else _starts([new] * 3, cuda)
    out, lse = cache.attend(q, seq, table, q_starts=starts, want_lse=True)
    _check(cache, table, lens, [new] * 3, q, out, lse)


@pytest.mark.parametrize("new", [1, 4, 100])
def test_sequences_that_share_their_first_pages(cuda, new):
    """A common prompt: several tables name the same pages."""
    lens = [256 + new, 300 + new, 256 + new]
    cache, table = _pages(cuda, lens, 32, 2, 128, new)
    table[1:, :8] = table[0, :8]
    q = _q(cuda, 3 * new, 8, 128, 9)
    seq, starts = torch.tensor(lens, dtype=torch.int32, device=cuda), None if new == 1 else _starts([new] * 3, cuda)
    out, lse = cache.attend(q, seq, table, q_starts=starts, want_lse=True)
    _check(cache, table, lens, [new] * 3, q, out, lse)


@pytest.mark.parametrize("d,ps,news,olds", [(128, 64, [2300, 1500], [0, 300]), (64, 16, [1900, 40, 700], [100, 2000, 0]), (128, 128, [1000] * 12, [200] * 12)])
def test_long_prompts(cuda, d, ps, news, olds):
    """More row tiles than fit on the GPU at once, each with many key tiles."""
    from oxicuda_b200 import _lib as L
    lens = [n + o for n, o in zip(news, olds)]
    cache, table = _pages(cuda, lens, ps, 4, d, len(lens))
    q = _q(cuda, sum(news), 16, d, ps)
    out, lse = cache.attend(q, torch.tensor(lens, dtype=torch.int32, device=cuda), table, q_starts=_starts(news, cuda), want_lse=True)
    L.default_handle().check()
    _check(cache, table, lens, news, q, out, lse)


@pytest.mark.parametrize("new,old", [(1, 9000), (2, 9000), (5, 9000), (40, 9000), (130, 6000)])
def test_long_keys_of_few_rows(cuda, new, old):
    """Keys dealt to the CTAs of a cluster, in every number of them that a batch of this kind meets."""
    for seqs in (1, 3, 6):
        lens = [old + new + 64 * i for i in range(seqs)]
        cache, table = _pages(cuda, lens, 64, 4, 128, seqs)
        q = _q(cuda, seqs * new, 8, 128, new)
        seq, starts = torch.tensor(lens, dtype=torch.int32, device=cuda), None if new == 1 else _starts([new] * seqs, cuda)
        out, lse = cache.attend(q, seq, table, q_starts=starts, want_lse=True)
        _check(cache, table, lens, [new] * seqs, q, out, lse)


@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("jump", [3, 9, 25])
@pytest.mark.parametrize("new", [1, 150])
def test_pages_of_different_sizes(cuda, ps, jump, new):
    """Neighbouring pages whose scales lie 2^3 to 2^25 apart, with rows whose weight falls on a page of the small kind."""
    lens = [640, 333 + new]
    cache, table = _pages(cuda, lens, ps, 2, 128, jump + ps, spread=0, jump=jump)
    cache.k_scales[cache.k_scales != 255] = 120            # keys of one size: the scores stay moderate
    news = [new, new]
    q = _q(cuda, 2 * new, 8, 128, jump)
    out = cache.attend(q, torch.tensor(lens, dtype=torch.int32, device=cuda), table, q_starts=None if new == 1 else _starts(news, cuda))
    _check(cache, table, lens, news, q, out)
    # values of the large pages set to 0 within the codes: what is left is the small pages' part alone
    small = cache.v_scales < 120 + jump
    cache.v_codes[~small & (cache.v_scales != 255)] = 0
    out = cache.attend(q, torch.tensor(lens, dtype=torch.int32, device=cuda), table, q_starts=None if new == 1 else _starts(news, cuda))
    for b, n in enumerate(lens):                           # the stale slots of the cleared pages are zeros now; they stay unread all the same
        assert torch.isfinite(out).all()
    _check(cache, table, lens, news, q, out)


@pytest.mark.parametrize("new", [1, 140])
def test_scale_argument_and_large_scores(cuda, new):
    lens = [900]
    cache, table = _pages(cuda, lens, 64, 2, 64, 4)
    for scale, size in ((1.0, 0.05), (-0.125, 1.0), (0.0, 1.0), (0.125, 30.0)):
        q = _q(cuda, new, 6, 64, 5, size)
        out, lse = cache.attend(q, torch.tensor(lens, dtype=torch.int32, device=cuda), table, q_starts=_starts([new], cuda), scale=scale, want_lse=True)
        _check(cache, table, lens, [new], q, out, lse, scale=scale)


@pytest.mark.parametrize("new", [1, 130])
def test_non_finite_queries_stay_in_their_row(cuda, new):
    lens = [70 + new]
    cache, table = _pages(cuda, lens, 16, 1, 128, 8)
    q = _q(cuda, new, 4, 128, 8)
    seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
    clean, clse = cache.attend(q, seq, table, q_starts=_starts([new], cuda), want_lse=True)
    q[0, 1, 5], q[new - 1, 2, 127] = float("nan"), float("inf")
    out, lse = cache.attend(q, seq, table, q_starts=_starts([new], cuda), want_lse=True)
    keep = torch.ones(new, 4, dtype=torch.bool, device=cuda)
    keep[0, 1] = keep[new - 1, 2] = False
    assert torch.isnan(out[~keep]).all() and torch.isnan(lse[~keep]).all()
    assert torch.equal(out[keep], clean[keep]) and torch.equal(lse[keep], clse[keep])


def test_rows_outside_every_sequence_and_out_argument(cuda):
    """A padded batch: rows behind the last sequence, and those of sequences of no tokens, are left as they were."""
    news, lens = [3, 0, 40], [10, 5, 90]
    cache, table = _pages(cuda, lens, 16, 2, 64, 12)
    q = _q(cuda, 60, 4, 64, 1)
    out = torch.full((60, 4, 64), 7.0, dtype=torch.bfloat16, device=cuda)
    got = cache.attend(q, torch.tensor(lens, dtype=torch.int32, device=cuda), table, q_starts=_starts(news, cuda), out=out)
    assert got is out and (out[43:] == 7).all()
    _check(cache, table, lens, news, q, out)
    starts = torch.tensor([5, 8, 8, 48], dtype=torch.int32, device=cuda)               # rows in front of the first one too
    out.fill_(7.0)
    cache.attend(q, torch.tensor(lens, dtype=torch.int32, device=cuda), table, q_starts=starts, out=out)
    assert (out[:5] == 7).all() and (out[48:] == 7).all()
    _check(cache, table, lens, news, q, out, r0s=[5, 8, 8])


def test_impossible_sequences_and_bad_pages_are_reported(cuda):
    from oxicuda_b200 import _lib as L
    lens = [40, 50, 60, 70]
    cache, table = _pages(cuda, lens, 16, 2, 128, 14)
    h = L.default_handle()
    q = _q(cuda, 4, 8, 128, 3)
    seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
    good = cache.attend(q, seq, table)
    bad = seq.clone()
    bad[1], bad[2] = 0, 1 << 30                                                       # no token, and more than the table holds
    out = torch.full_like(good, 7.0)
    cache.attend(q, bad, table, out=out)
    with pytest.raises(L.InvalidDimension):
        h.check()
    assert (out[1:3] == 7).all() and torch.equal(out[0], good[0]) and torch.equal(out[3], good[3])
    for starts in ([0, 1, 0, 3, 4], [0, 1, 2, 3, 9], [-1, 1, 2, 3, 4]):
        out.fill_(7.0)
        cache.attend(q, seq, table, q_starts=torch.tensor(starts, dtype=torch.int32, device=cuda), out=out)
        with pytest.raises(L.InvalidDimension):
            h.check()
    t2 = table.clone()
    t2[0, 1], t2[3, 0] = cache.num_pages, -5
    for starts in (None, torch.arange(5, dtype=torch.int32, device=cuda)):
        out = cache.attend(q, seq, t2, q_starts=starts)
        with pytest.raises(L.InvalidArgument):
            h.check()
        assert torch.equal(out[1], good[1]) or starts is not None
        assert torch.isfinite(out).all()
    h.check()


def test_strided_queries_and_results_do_not_depend_on_neighbours(cuda):
    lens = [300, 17]
    cache, table = _pages(cuda, lens, 32, 2, 128, 19)
    wide = torch.randn(2, 3 * 8 * 128, device=cuda).to(torch.bfloat16)
    q = wide[:, 1024: 2048].view(2, 8, 128)                                           # the middle of a fused projection's rows
    seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
    a = cache.attend(q, seq, table)
    assert torch.equal(a, cache.attend(q.contiguous(), seq, table))
    assert torch.equal(a[1:], cache.attend(q[1:], seq[1:], table[1:].contiguous()))
    odd = torch.empty(2 * 8 * 128 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(2, 8, 128)
    odd.copy_(q)
    assert torch.equal(a, cache.attend(odd, seq, table))
    _check(cache, table, lens, [1, 1], q, a)


def test_long_cache_and_offsets_beyond_32_bits(cuda):
    """Pages whose codes lie more than 2^32 bytes into the pool."""
    from oxicuda_b200.kv_cache import PagedFp8KvCache
    kvh, ps, d, num = 8, 128, 128, 40000                                              # 5.2 GB of codes each for K and V
    codes = [torch.full((num, kvh, ps, d), 0x7F, dtype=torch.uint8, device=cuda) for _ in range(2)]
    scales = [torch.full((num, kvh), 120, dtype=torch.uint8, device=cuda) for _ in range(2)]
    cache = PagedFp8KvCache(*codes, *scales)
    lens, news = [20000, 700], [1, 130]
    table = torch.full((2, 160), -1, dtype=torch.int32, device=cuda)
    table[0, :157] = torch.arange(num - 157, num, dtype=torch.int32, device=cuda)
    table[1, :6] = torch.arange(33000, 33006, dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(2)
    for c in codes:
        for lo, hi in ((num - 157, num), (33000, 33006)):
            c[lo:hi] = (100 * torch.randn(hi - lo, kvh, ps, d, device=cuda, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    q = _q(cuda, 131, 16, d, 6)
    seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
    out = cache.attend(q, seq, table, q_starts=_starts(news, cuda))
    _check(cache, table, lens, news, q, out)
    one = cache.attend(q[:2], seq, table)
    _check(cache, table, lens, [1, 1], q, one)
    k = torch.randn(2, kvh, d, device=cuda, generator=g).to(torch.bfloat16)
    cache.append(k, k, seq, table)
    v = cache.v_codes[num - 1, :, 19999 % ps].view(torch.float8_e4m3fn).float() * torch.exp2(cache.v_scales[num - 1].float() - 127)[:, None]
    assert ((v - k[0].float()).abs() <= 2.0 ** -4 * k[0].float().abs() + 2.0 ** -10 * torch.exp2(cache.v_scales[num - 1].float() - 127)[:, None]).all()


def test_two_streams_and_two_graphs(cuda):
    lens = [[3000, 70], [900, 44, 5], [200]]
    news = [[1, 1], [1, 1, 1], [180]]
    sets = []
    for i, (n, m) in enumerate(zip(lens, news)):
        cache, table = _pages(cuda, n, 16, 2, 128, i)
        sets.append((cache, table, _q(cuda, sum(m), 8, 128, i), torch.tensor(n, dtype=torch.int32, device=cuda), None if max(m) == 1 else _starts(m, cuda)))
    run = lambda s: s[0].attend(s[2], s[3], s[1], q_starts=s[4])
    want = [run(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(4):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(run(s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(run(s))
        graphs.append(gr)
    for o in outs:
        o.zero_()
    for st, gr in zip(streams, graphs):
        with torch.cuda.stream(st):
            gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    # lengths are read on the device: a captured step follows them
    s = sets[0]
    s[3].copy_(torch.tensor([2500, 33], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    _check(s[0], s[1], [2500, 33], [1, 1], s[2], outs[0])


# ---- append -----------------------------------------------------------------------------------------------------------
def _encode(x):
    """The nearest E4M3 code of x (64 bits), ties to even, at most 448 in size, by search over all codes."""
    table = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().to(x.device)
    a = x.abs().clamp(max=448.0)
    hi = torch.searchsorted(table, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - table[lo], table[hi] - a
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (pick + torch.where(torch.signbit(x), 128, 0)).to(torch.uint8)


def _append_ref(codes, scales, x, lens, news, table, ps):
    """By definition, one page and head at a time; codes and scales are changed in place."""
    r0 = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        first = n - m
        for i in range(first // ps, (n - 1) // ps + 1) if m else []:
            pg, lo, hi = int(table[b, i]), max(first, i * ps), min(n, (i + 1) * ps)
            for h in range(codes.shape[1]):
                new = x[r0 + lo - first: r0 + hi - first, h].double()
                top = float(new[torch.isfinite(new)].abs().max()) if torch.isfinite(new).any() else 0.0
                e = -50
                while top > 448.0 * 2.0 ** e and e < 119:
                    e += 1
                if lo > i * ps:
                    old = int(scales[pg, h]) - 127
                    e = max(e, old)
                    was = codes[pg, h, : lo - i * ps].view(torch.float8_e4m3fn).double() * 2.0 ** (old - e)
                    codes[pg, h, : lo - i * ps] = _encode(was)
                scales[pg, h] = e + 127
                y = torch.nan_to_num(new * 2.0 ** -e, nan=0.0, posinf=448.0, neginf=-448.0)
                codes[pg, h, lo - i * ps: hi - i * ps] = _encode(y)
        r0 += m


@pytest.mark.parametrize("d,ps", [(64, 16), (128, 16), (128, 32), (128, 64), (64, 128)])
@pytest.mark.parametrize("news,olds", [([1], [0]), ([1, 1, 1, 1], [0, 5, 16, 700]), ([3, 0, 20], [0, 9, 15]), ([130, 1, 17], [3, 31, 128]), ([300], [0])])
def test_append_bit_for_bit(cuda, d, ps, news, olds):
    lens = [n + o for n, o in zip(news, olds)]
    g = torch.Generator(device=cuda).manual_seed(sum(lens) + d)
    for size in (0.01, 1.0, 3e4):                          # smaller than what the pages hold, alike, and far larger (codes move)
        cache, table = _pages(cuda, lens, ps, 3, d, sum(lens))
        k = (size * torch.randn(sum(news), 3, d, device=cuda, generator=g)).to(torch.bfloat16)
        v = (size * torch.randn(sum(news), 3, d, device=cuda, generator=g)).to(torch.bfloat16)
        v[0, 1] = 0
        k[-1, 2, 0] = 1.75 * 2 ** 5                        # exactly 448 * 2^-3: the largest code under that scale
        want = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
        _append_ref(want[0], want[1], k, lens, news, table, ps)
        _append_ref(want[2], want[3], v, lens, news, table, ps)
        starts = None if news == [1] * len(news) else _starts(news, cuda)
        cache.append(k, v, torch.tensor(lens, dtype=torch.int32, device=cuda), table, q_starts=starts)
        for name, w, got in zip(("k", "k_scales", "v", "v_scales"), want, (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)):
            assert torch.equal(w, got), (name, size)


def test_append_token_by_token_and_its_own_repetition(cuda):
    """Tokens appended one at a time meet growing scales; appending the last one again changes nothing."""
    from oxicuda_b200.kv_cache import PagedFp8KvCache
    g = torch.Generator(device=cuda).manual_seed(31)
    n, ps, d = 40, 16, 64
    x = torch.randn(n, 2, d, device=cuda, generator=g) * torch.logspace(-3, 2, n, device=cuda)[:, None, None]
    x = x.to(torch.bfloat16)
    cache = PagedFp8KvCache.empty(4, ps, 2, d, cuda)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device=cuda)
    want = [t.clone() for t in (cache.k_codes, cache.k_scales)]
    for i in range(n):
        cache.append(x[i: i + 1], x[i: i + 1], torch.tensor([i + 1], dtype=torch.int32, device=cuda), table)
        _append_ref(want[0], want[1], x[i: i + 1], [i + 1], [1], table, ps)
    assert torch.equal(cache.k_codes, want[0]) and torch.equal(cache.k_scales, want[1])
    assert torch.equal(cache.k_codes, cache.v_codes) and torch.equal(cache.k_scales, cache.v_scales)
    cache.append(x[-1:], x[-1:], torch.tensor([n], dtype=torch.int32, device=cuda), table)
    assert torch.equal(cache.k_codes, want[0]) and torch.equal(cache.k_scales, want[1])


def test_append_of_non_finite_values_and_extremes(cuda):
    from oxicuda_b200 import _lib as L
    from oxicuda_b200.kv_cache import PagedFp8KvCache
    h = L.default_handle()
    table = torch.tensor([[1]], dtype=torch.int32, device=cuda)
    x = torch.zeros(3, 1, 64, dtype=torch.bfloat16, device=cuda)
    x[0, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 2.0])
    cache = PagedFp8KvCache.empty(2, 16, 1, 64, cuda)
    cache.append(x, x, torch.tensor([3], dtype=torch.int32, device=cuda), table, q_starts=torch.tensor([0, 3], dtype=torch.int32, device=cuda))
    with pytest.raises(L.NonFiniteFp8):
        h.check()
    want = [t.clone() for t in (cache.k_codes, cache.k_scales)]
    _append_ref(want[0], want[1], x, [3], [3], table, 16)
    assert torch.equal(cache.k_codes, want[0]) and torch.equal(cache.k_scales, want[1])
    for top in (3.3e38, 1e-38, 0.0):
        x = torch.full((1, 1, 64), top, dtype=torch.bfloat16, device=cuda)
        cache = PagedFp8KvCache.empty(2, 16, 1, 64, cuda)
        cache.append(x, x, torch.tensor([1], dtype=torch.int32, device=cuda), table)
        want = [torch.zeros_like(cache.k_codes), torch.full_like(cache.k_scales, 127)]
        _append_ref(want[0], want[1], x, [1], [1], table, 16)
        assert torch.equal(cache.k_codes, want[0]) and torch.equal(cache.k_scales, want[1])
    h.check()


def test_append_leaves_out_what_cannot_be(cuda):
    from oxicuda_b200 import _lib as L
    lens = [40, 50, 60]
    cache, table = _pages(cuda, lens, 16, 2, 64, 41)
    h = L.default_handle()
    x = torch.randn(3, 2, 64, device=cuda).to(torch.bfloat16)
    before = [t.clone() for t in (cache.k_codes, cache.k_scales)]
    t2 = table.clone()
    t2[1, 3] = cache.num_pages
    cache.append(x, x, torch.tensor([0, 50, 1 << 29], dtype=torch.int32, device=cuda), t2)
    with pytest.raises((L.InvalidDimension, L.InvalidArgument)):
        h.check()
    assert torch.equal(cache.k_codes, before[0]) and torch.equal(cache.k_scales, before[1])
    cache.append(x, x, torch.tensor(lens, dtype=torch.int32, device=cuda), table, q_starts=torch.tensor([0, 2, 1, 7], dtype=torch.int32, device=cuda))
    with pytest.raises(L.InvalidDimension):
        h.check()
    h.check()


def test_append_takes_views_of_a_projection(cuda):
    lens, news = [100, 33], [20, 3]
    g = torch.Generator(device=cuda).manual_seed(4)
    qkv = torch.randn(23, (8 + 2 * 2) * 64, device=cuda, generator=g).to(torch.bfloat16)
    k, v = qkv[:, 512: 640].view(23, 2, 64), qkv[:, 640:].view(23, 2, 64)
    a, table = _pages(cuda, lens, 16, 2, 64, 5)
    b, _ = _pages(cuda, lens, 16, 2, 64, 5)
    seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
    a.append(k, v, seq, table, q_starts=_starts(news, cuda))
    b.append(k.contiguous(), v.contiguous(), seq, table, q_starts=_starts(news, cuda))
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        assert torch.equal(getattr(a, name), getattr(b, name))


def test_append_and_attend_together(cuda):
    """Prefill, then decode steps, as a runner makes them: every step's attention sees what the steps before it stored."""
    from oxicuda_b200.kv_cache import PagedFp8KvCache
    g = torch.Generator(device=cuda).manual_seed(51)
    kvh, group, d, ps = 2, 4, 128, 16
    cache = PagedFp8KvCache.empty(40, ps, kvh, d, cuda)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(2, 20).to(cuda)
    lens = [0, 0]
    for news in ([37, 150], [1, 1], [1, 1], [4, 2], [1, 1]):
        lens = [a + b for a, b in zip(lens, news)]
        rows = sum(news)
        k, v = [torch.randn(rows, kvh, d, device=cuda, generator=g).to(torch.bfloat16) for _ in range(2)]
        q = torch.randn(rows, kvh * group, d, device=cuda, generator=g).to(torch.bfloat16)
        seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
        starts = None if max(news) == 1 else _starts(news, cuda)
        cache.append(k, v, seq, table, q_starts=starts)
        out, lse = cache.attend(q, seq, table, q_starts=starts, want_lse=True)
        _check(cache, table, lens, news, q, out, lse)
