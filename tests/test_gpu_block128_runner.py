"""GPU: the decoder of model_runner.py with recipe="block128": every stage of every layer recomputed in 64 bits from the runner's own inputs
of that stage, prefill and decode steps over a ragged batch, and against plain fp32 end to end."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _dense(lin):
    s = lin.scales.double().repeat_interleave(128, 0)[: lin.out_features].repeat_interleave(128, 1)[:, : lin.in_features]
    return lin.codes.view(torch.float8_e4m3fn).double() * s


def _q128(t):
    """[rows, cols] -> the values of E4M3 codes with a scale per 128 columns."""
    rows, cols = t.shape
    nb = -(-cols // 128)
    b = torch.nn.functional.pad(t, (0, nb * 128 - cols)).view(rows, nb, 128)
    s = b.abs().amax(dim=2, keepdim=True) / 448.0
    s = torch.where(s > 0, s, torch.ones_like(s))
    return ((b / s).float().to(torch.float8_e4m3fn).double() * s).reshape(rows, -1)[:, :cols]


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _rms(x, g, eps):
    return x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + eps) * g.double()


def _rope(runner, t, positions):
    d = t.shape[-1]
    ang = positions.to(torch.float32)[:, None] * runner.inv_freq[None, :]
    cos, sin = ang.cos()[:, None, :].double(), ang.sin()[:, None, :].double()
    a, b = t[..., : d // 2], t[..., d // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)


def _cached(cache, table, n, which):
    codes, scales = (cache.k_codes, cache.k_scales) if which == "k" else (cache.v_codes, cache.v_scales)
    pages = torch.tensor(table[: -(-n // cache.page_size)], device=codes.device)
    v = codes[pages].view(torch.float8_e4m3fn).double() * torch.exp2(scales[pages].double() - 127)[:, :, None, None]
    return v.permute(0, 2, 1, 3).reshape(-1, cache.n_kv_heads, cache.head_dim)[:n]


def _stage_checks(runner, trace, positions, seqs):
    """seqs: (row0, row1, cached tokens with these, block table).  Norms of the differences: a bf16 result is off by 2^-9 of itself in the
    mean, so 4e-3 holds a stage that ends in bf16; an E4M3 rounding in front of it re-rolls few codes, those within 1e-6 of a boundary."""
    cfg = runner.cfg
    nq, nkv, d = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
    bf = lambda t: t.to(torch.bfloat16).double()
    res = torch.zeros_like(trace[0]["res_attn"]).double()
    for layer, t in zip(runner.layers, trace):
        tokens = t["qkv"].shape[0]
        res = bf((res + t["x_in"].double()).float())
        assert torch.equal(t["res_attn"].double(), res)
        assert _rel(t["qkv"], _q128(_rms(res, layer.g_attn, cfg.eps)) @ _dense(layer.qkv).t()) <= 4e-3
        qkv = t["qkv"].double()
        q = bf(_rope(runner, qkv[:, : nq * d].reshape(tokens, nq, d), positions))
        k = bf(_rope(runner, qkv[:, nq * d: (nq + nkv) * d].reshape(tokens, nkv, d), positions))
        v = qkv[:, (nq + nkv) * d:].reshape(tokens, nkv, d)
        attn = torch.empty(tokens, nq, d, dtype=torch.float64, device=res.device)
        for r0, r1, n, table in seqs:
            kc, vc = _cached(layer.cache, table, n, "k"), _cached(layer.cache, table, n, "v")
            # what the step stored: E4M3 under a scale that the page may share with larger tokens (half a step, 2^-4; 2^-10 of the scale below)
            for mine, stored, scales in ((k, kc, layer.cache.k_scales), (v, vc, layer.cache.v_scales)):
                s = torch.exp2(scales.double() - 127)[torch.tensor(table, device=res.device)].repeat_interleave(cfg.block_size, 0)[n - (r1 - r0): n]
                assert ((stored[n - (r1 - r0):] - mine[r0:r1]).abs() <= torch.maximum(2.0 ** -4 * mine[r0:r1].abs(), 2.0 ** -10 * s[..., None])).all()
            kk, vv = kc.repeat_interleave(nq // nkv, dim=1), vc.repeat_interleave(nq // nkv, dim=1)
            sc = torch.einsum("qhd,khd->hqk", q[r0:r1], kk) / math.sqrt(d)
            j = torch.arange(n, device=res.device)
            sc = sc.masked_fill((j[None] > (n - (r1 - r0) + torch.arange(r1 - r0, device=res.device))[:, None])[None], -math.inf)
            attn[r0:r1] = torch.einsum("hqk,khd->qhd", torch.softmax(sc, dim=-1), vv)
        assert _rel(t["attn"], attn) <= 4e-3
        assert _rel(t["o_out"], _q128(t["attn"].double().reshape(tokens, nq * d)) @ _dense(layer.o).t()) <= 1e-2     # bf16 inputs meet exact E4M3 ties
        res = bf((res + t["o_out"].double()).float())
        assert torch.equal(t["res_mlp"].double(), res)
        assert _rel(t["gu"], _q128(_rms(res, layer.g_mlp, cfg.eps)) @ _dense(layer.gate_up).t()) <= 4e-3
        g, u = t["gu"].double()[:, : cfg.ffn], t["gu"].double()[:, cfg.ffn:]
        assert _rel(t["mlp_out"], _q128(g * torch.sigmoid(g) * u) @ _dense(layer.down).t()) <= 4e-3


def _plain_logits(runner, ids, positions, rows):
    """fp32 statement over whole sequences with the same dequantized weights, no quantized activations or cache."""
    cfg = runner.cfg
    nq, nkv, d = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
    res = runner.embed[ids.long()].double()
    for layer in runner.layers:
        qkv = _rms(res, layer.g_attn, cfg.eps) @ _dense(layer.qkv).t()
        n = qkv.shape[0]
        q, k = _rope(runner, qkv[:, : nq * d].reshape(n, nq, d), positions), _rope(runner, qkv[:, nq * d: (nq + nkv) * d].reshape(n, nkv, d), positions)
        v = qkv[:, (nq + nkv) * d:].reshape(n, nkv, d)
        attn = torch.empty(n, nq, d, dtype=torch.float64, device=res.device)
        for r0, r1 in rows:
            s = torch.einsum("qhd,khd->hqk", q[r0:r1], k[r0:r1].repeat_interleave(nq // nkv, dim=1)) / math.sqrt(d)
            s = s.masked_fill(torch.triu(torch.ones(r1 - r0, r1 - r0, dtype=torch.bool, device=res.device), 1)[None], -math.inf)
            attn[r0:r1] = torch.einsum("hqk,khd->qhd", torch.softmax(s, dim=-1), v[r0:r1].repeat_interleave(nq // nkv, dim=1))
        res = res + attn.reshape(n, nq * d) @ _dense(layer.o).t()
        gu = _rms(res, layer.g_mlp, cfg.eps) @ _dense(layer.gate_up).t()
        g, u = gu[:, : cfg.ffn], gu[:, cfg.ffn:]
        res = res + (g * torch.sigmoid(g) * u) @ _dense(layer.down).t()
    return _rms(res, runner.g_final, cfg.eps) @ _dense(runner.lm_head).t()


@pytest.mark.parametrize("head_dim,page", [(64, 16), (128, 32)])
def test_prefill_and_decode_stage_by_stage(cuda, head_dim, page):
    from oxicuda_b200.model_runner import LlamaConfig, QuantizedLlamaRunner
    cfg = LlamaConfig(head_dim=head_dim, block_size=page, recipe="block128")
    runner = QuantizedLlamaRunner(cfg, cuda, seed=9)
    rng = np.random.default_rng(5)
    lens = [5, 23, 70]
    prompts = [rng.integers(0, cfg.vocab_size, n).tolist() for n in lens]
    tables = [[9, 1], [2, 30, 4], [5, 6, 50, 8, 21]]
    starts = [0, 5, 28, 98]
    runner.trace = []
    logits = runner.prefill([t for p in prompts for t in p], starts, tables)
    pos = torch.cat([torch.arange(n, device=cuda) for n in lens])
    _stage_checks(runner, runner.trace, pos, [(starts[i], starts[i + 1], lens[i], tables[i]) for i in range(3)])
    for step in range(2):
        nxt = [int(np.argmax(row)) for row in logits]
        runner.trace = []
        logits = runner.decode(nxt, tables, lens)
        pos = torch.tensor(lens, device=cuda)
        lens = [n + 1 for n in lens]
        for p, t in zip(prompts, nxt):
            p.append(t)
        _stage_checks(runner, runner.trace, pos, [(i, i + 1, lens[i], tables[i]) for i in range(3)])
    runner.trace = None
    # end to end: each E4M3 rounding of activations or cache adds noise of 3 mantissa bits (3.6 % rms at most) to a stage's input; the bound is
    # the one that the per-token recipe's runner is held to
    st = [0]
    for n in lens:
        st.append(st[-1] + n)
    ids = torch.tensor([t for p in prompts for t in p], device=cuda)
    pos = torch.cat([torch.arange(n, device=cuda) for n in lens])
    ref = _plain_logits(runner, ids, pos, [(st[i], st[i + 1]) for i in range(3)])[[s - 1 for s in st[1:]]]
    assert _rel(torch.tensor(logits, device=cuda), ref) <= 0.12


def test_runner_contract_and_refusals(cuda):
    from oxicuda_b200 import _lib
    from oxicuda_b200.model_runner import EmptyBatch, LlamaConfig, QuantizedLlamaRunner
    runner = QuantizedLlamaRunner(LlamaConfig(n_layers=1, recipe="block128"), cuda)
    with pytest.raises(EmptyBatch):
        runner.decode([], [], [])
    with pytest.raises(EmptyBatch):
        runner.prefill([], [0], [])
    with pytest.raises(_lib.DimensionMismatch):                # a sequence longer than its block table
        runner.decode([1], [[0]], [16])
    with pytest.raises(_lib.InvalidArgument):                  # a block that the cache does not have
        runner.decode([1], [[64]], [3])
    for bad in (LlamaConfig(recipe="block64"), LlamaConfig(recipe="block128", n_heads=1, n_kv_heads=1)):
        with pytest.raises(_lib.InvalidConfig):
            QuantizedLlamaRunner(bad, cuda)
    with pytest.raises(_lib.UnsupportedOperation):
        QuantizedLlamaRunner(LlamaConfig(recipe="block128", block_size=24), cuda)


def test_padded_block_tables(cuda):
    """Tables as a server keeps them, padded to one width, give the logits of exact ones."""
    from oxicuda_b200.model_runner import LlamaConfig, QuantizedLlamaRunner
    cfg = LlamaConfig(n_layers=1, recipe="block128")
    got = []
    for pad in ([], [-1] * 9):
        runner = QuantizedLlamaRunner(cfg, cuda, seed=4)
        tables = [[9, 1, 3] + pad, [2, 30] + pad]
        got.append([runner.prefill(list(range(40)), [0, 33, 40], tables), runner.decode([5, 6], tables, [33, 7])])
    assert got[0] == got[1]
