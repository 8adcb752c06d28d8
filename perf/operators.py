"""Cases of the block-128 FP8 decoder path, with each operator's plain form in elementary torch operations.

Five operators, as one decoder layer uses them one after the other:
  norm      residual add + RMSNorm + E4M3 codes with a scale per 128 columns (feeds the q|k|v and gate|up projections)
  gemm      the FP8 product over those operands: a scale per (row, 128 columns) and per 128 x 128 weight block
  append    new keys and values into a paged cache of E4M3 codes with one power-of-two scale per (page, kv head)
  attend    attention that reads those pages
  swiglu    silu(gate) * up + E4M3 codes with a scale per 128 columns (feeds the down projection)
"""
import math

import torch

own = False

E4M3_MAX = 448.0
MIN_EXP, MAX_EXP = -50, 119           # exponents of the cache's scales


def listed():
    return [
        # one token through a 4096 -> 14336 projection: decode, latency and the weights' bytes count
        {"name": "gemm decode 1 token", "op": "gemm", "m": 1, "n": 14336, "k": 4096, "out": "bf16"},
        # a batch of decoding sequences (ragged count) through 8192 -> 8192 + 2 x 1024 rows of q|k|v
        {"name": "gemm decode 53 tokens", "op": "gemm", "m": 53, "n": 10240, "k": 8192, "out": "bf16"},
        # a prompt chunk of 4096 tokens through the 28672 -> 8192 down projection: the largest product of a layer
        {"name": "gemm prefill 4096 tokens", "op": "gemm", "m": 4096, "n": 8192, "k": 28672, "out": "bf16"},
        # a few decoding sequences in front of a 4096-wide projection
        {"name": "norm 7 tokens", "op": "norm", "rows": 7, "cols": 4096, "residual": True, "y": False},
        # a prompt chunk in front of an 8192-wide projection
        {"name": "norm 4096 tokens", "op": "norm", "rows": 4096, "cols": 8192, "residual": True, "y": False},
        # the activation between the projections, one decoding sequence (the two halves of one row)
        {"name": "swiglu 1 token", "op": "swiglu", "rows": 1, "cols": 14336},
        # the same for a prompt chunk, ragged row count
        {"name": "swiglu 2047 tokens", "op": "swiglu", "rows": 2047, "cols": 28672},
        # one new token for each of 48 sequences
        {"name": "append decode", "op": "append", "seqs": 48, "new": 1, "old": 700, "kv_heads": 8, "head_dim": 128, "page": 16},
        # prompts of about 1500 tokens behind a cached prefix that ends inside a page
        {"name": "append prefill", "op": "append", "seqs": 6, "new": 1500, "old": 37, "kv_heads": 8, "head_dim": 128, "page": 64},
        # a single short conversation: one token against 333 cached ones, where latency counts
        {"name": "attend decode short", "op": "attend", "seqs": 1, "new": 1, "old": 332, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 16, "window": 0, "lse": False},
        # a serving batch: one token each against about 8000 cached ones
        {"name": "attend decode batch", "op": "attend", "seqs": 32, "new": 1, "old": 8200, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 64, "window": 0, "lse": False},
        # prompts of about 4000 tokens, part of them cached already, with the log-sum-exp that a later merge needs
        {"name": "attend prefill", "op": "attend", "seqs": 2, "new": 3900, "old": 150, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 64, "window": 0, "lse": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "norm", "swiglu", "append", "attend", "attend"])
    if op == "gemm":
        n = _log(rng, 64, 28672)
        k = 16 * _log(rng, 8, 1792)                    # rows of codes are 16-byte aligned; the last block of 128 may be short
        m = min(_log(rng, 1, 4096), max(1, 4096 * 8192 * 28672 // (n * k)))
        return {"op": "gemm", "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "bf16", "f32"])}
    if op == "norm":
        return {"op": "norm", "rows": _log(rng, 1, 4096), "cols": 8 * _log(rng, 16, 1024), "residual": rng.random() < 0.7, "y": rng.random() < 0.3}
    if op == "swiglu":
        return {"op": "swiglu", "rows": _log(rng, 1, 2047), "cols": 8 * _log(rng, 16, 3584)}
    kv_heads = rng.choice([1, 2, 4, 8])
    head_dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        new = rng.choice([1, 1, _log(rng, 2, 1500)])
        seqs = max(1, min(_log(rng, 1, 64), 9000 // new))
        return {"op": "append", "seqs": seqs, "new": new, "old": _log(rng, 1, 1000), "kv_heads": kv_heads, "head_dim": head_dim, "page": page}
    heads = kv_heads * rng.choice([1, 4, 4, 7, 8])
    if rng.random() < 0.5:                             # decode, now and then with a few draft tokens
        new = rng.choice([1, 1, 1, 4])
        old = _log(rng, 1, 16000)
        seqs = max(1, min(_log(rng, 1, 64), 260000 // (old + new)))
    else:
        new = _log(rng, 16, 3900)
        old = _log(rng, 1, 2000)
        seqs = max(1, min(_log(rng, 1, 8), 32 * 4050 * 4050 // (heads * new * (old + new))))
    return {"op": "attend", "seqs": seqs, "new": new, "old": old, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "window": rng.choice([0, 0, 0, _log(rng, 32, 4000)]), "lse": rng.random() < 0.3}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _activations(g, rows, cols):
    """bf16 activations whose channels differ in size, a few of them by much, as the residual stream of a decoder has them."""
    x = _randn(g, rows, cols) * torch.exp(0.5 * _randn(g, cols))
    x[:, torch.randint(0, cols, (max(1, cols // 512),), device="cuda", generator=g)] *= 12.0
    return x.to(torch.bfloat16)


def _blocks(x):
    """[rows, cols] -> [rows, ceil(cols / 128), 128], filled up with zeros."""
    rows, cols = x.shape
    nb = (cols + 127) // 128
    return torch.nn.functional.pad(x, (0, nb * 128 - cols)).view(rows, nb, 128)


def _quantize(y):
    """One scale per (row, 128 columns): absmax / 448, 1 for a block of zeros; codes round to nearest even."""
    b = _blocks(y)
    amax = b.abs().amax(dim=2)
    s = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
    q = (b / s[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return q.reshape(y.shape[0], -1)[:, : y.shape[1]].to(torch.float32).to(torch.float8_e4m3fn).contiguous(), s


def _lengths(case):
    """New and cached tokens of each sequence: ragged below the case's figures, the first sequence with exactly those."""
    g = torch.Generator().manual_seed(case["seqs"] * 31 + case["new"] + case["old"])
    u = torch.rand(2, case["seqs"], generator=g)
    new = torch.full((case["seqs"],), case["new"]) if case["new"] <= 4 else (case["new"] * (0.6 + 0.4 * u[0])).long().clamp(min=1)
    old = (case["old"] * (0.5 + 0.5 * u[1])).long()
    new[0], old[0] = case["new"], case["old"]
    return new.tolist(), old.tolist()


def _scale_exp(amax):
    """Smallest e with amax <= 448 * 2^e, within the range that the cache stores; the least for a block of zeros."""
    mant, e = torch.frexp(amax)
    e = e.to(torch.int32) - 9 + (mant > 0.875).to(torch.int32)
    return torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).clamp(MIN_EXP, MAX_EXP)


def _pow2(e):
    """2^e for e of -126 .. 127, exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "gemm":
        a, sa = _quantize(_activations(g, case["m"], case["k"]).float())
        n, k = case["n"], case["k"]
        nb, kb = (n + 127) // 128, (k + 127) // 128
        w = torch.empty(n, k, dtype=torch.float8_e4m3fn, device="cuda")
        sw = torch.empty(nb, kb, device="cuda")
        for r in range(0, n, 4096):                    # weights ~ N(0, 0.02), one scale per 128 x 128 block
            x = 0.02 * _randn(g, min(4096, n - r), k)
            t = torch.nn.functional.pad(x, (0, kb * 128 - k, 0, -x.shape[0] % 128))
            s = t.view(-1, 128, kb, 128).abs().amax(dim=(1, 3)) / E4M3_MAX
            full = s.repeat_interleave(128, 0)[: x.shape[0]].repeat_interleave(128, 1)[:, :k]
            w[r: r + x.shape[0]] = (x / full).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
            sw[r // 128: r // 128 + s.shape[0]] = s
        return {"op": op, "a": a.view(torch.uint8), "w": w.view(torch.uint8), "sa": sa, "sw": sw,
                "out": torch.bfloat16 if case["out"] == "bf16" else torch.float32}
    if op == "norm":
        x = _activations(g, case["rows"], case["cols"])
        return {"op": op, "x": x, "residual": _activations(g, case["rows"], case["cols"]) if case["residual"] else None,
                "gamma": (1.0 + 0.1 * _randn(g, case["cols"])).to(torch.bfloat16), "eps": 1e-5, "y": case["y"]}
    if op == "swiglu":
        return {"op": op, "gu": (1.5 * _randn(g, case["rows"], 2 * case["cols"])).to(torch.bfloat16)}
    new, old = _lengths(case)
    ps, kvh, d = case["page"], case["kv_heads"], case["head_dim"]
    total = [n + o for n, o in zip(new, old)]
    pages = [(t + ps - 1) // ps for t in total]
    width = max(pages) + 1
    num = sum(pages) + 3
    order = torch.randperm(num, generator=torch.Generator().manual_seed(int(seed) + 1)).tolist()
    table = [[-1] * width for _ in pages]
    at = 0
    for b, p in enumerate(pages):
        table[b][:p] = order[at: at + p]
        at += p
    st = {"op": op, "seq_lens": torch.tensor(total, dtype=torch.int32, device="cuda"), "table": torch.tensor(table, dtype=torch.int32, device="cuda"),
          "page": ps}
    rows = sum(new)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st["starts"] = None if case["new"] == 1 else torch.tensor(starts, dtype=torch.int32, device="cuda")
    codes, scales = [], []
    for _ in range(2):                                 # keys, then values: heads and pages of different sizes
        x = _randn(g, num, kvh, ps, d) * torch.exp(0.6 * _randn(g, 1, kvh, 1, 1)) * torch.exp(0.2 * _randn(g, num, 1, 1, 1))
        e = _scale_exp(x.abs().amax(dim=(2, 3)))
        codes.append((x * _pow2(-e)[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8))
        scales.append((e + 127).to(torch.uint8))
    # what a plan of the plain form keeps: the position of every new row, and of every key of every sequence in the pages
    st["plan"] = {"seq": torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda(),
                  "row": torch.cat([torch.arange(n) for n in new]).cuda(),
                  "pos": torch.cat([torch.arange(o, o + n) for n, o in zip(new, old)]).cuda(),
                  "old": torch.tensor(old, device="cuda"), "new": torch.tensor(new, device="cuda"), "max_new": max(new), "max_len": max(total)}
    st["k_codes"], st["v_codes"], st["k_scales"], st["v_scales"] = codes + scales
    if own:
        from oxicuda_b200.kv_cache import PagedFp8KvCache
        st["cache"] = PagedFp8KvCache(*codes, *scales)
    if op == "append":
        st["k"] = _activations(g, rows, kvh * d).view(rows, kvh, d)
        st["v"] = _randn(g, rows, kvh, d).to(torch.bfloat16)
    else:
        st["q"] = (1.3 * _randn(g, rows, case["heads"], d)).to(torch.bfloat16)
        st["window"], st["lse"] = case["window"], case["lse"]
    return st


# ---- plain forms ------------------------------------------------------------------------------------------------------
def _dense(codes, scales, rows_per):
    """Codes times their block scales, in 32 bits."""
    v = codes.view(torch.float8_e4m3fn).float()
    s = scales.repeat_interleave(128, 1)[:, : v.shape[1]]
    return v * (s if rows_per == 1 else s.repeat_interleave(rows_per, 0)[: v.shape[0]])


def _norm(s):
    x, res = s["x"].float(), s["residual"]
    if res is not None:
        res.copy_(res.float() + x)                     # the residual stream is updated in place, and the norm is of the stored sum
        x = res.float()
    y = x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + s["eps"]) * s["gamma"].float()
    codes, scales = _quantize(y)
    out = {"codes": codes, "scales": scales}
    if res is not None:
        out["residual"] = res
    if s["y"]:
        out["y"] = y.to(torch.bfloat16)
    return out


def _append_one(s, codes, scales, x):
    """Rows x [rows, heads, d] into their pages.  A page that held tokens before keeps them: its scale never shrinks, and when it grows
    its codes are encoded again under the new one."""
    p, ps = s["plan"], s["page"]
    page = s["table"].long()[p["seq"], p["pos"] // ps]
    slot = p["pos"] % ps
    num, kvh = scales.shape
    held = torch.zeros(num, dtype=torch.bool, device=x.device)
    at = p["old"] // ps                                # the page in which each sequence's first new token lies, if it holds old ones
    held[s["table"].long()[torch.arange(at.numel(), device=x.device), at]] = p["old"] % ps > 0
    amax = torch.zeros(num, kvh, device=x.device).index_reduce_(0, page, x.float().abs().amax(dim=2), "amax")
    touched = torch.zeros(num, dtype=torch.bool, device=x.device).index_fill_(0, page, True)
    was = scales.to(torch.int32) - 127
    e = torch.maximum(_scale_exp(amax), torch.where(held[:, None], was, torch.full_like(was, MIN_EXP)))
    e = torch.where(touched[:, None], e, was)
    grown = (held & touched)[:, None] & (e > was)
    # the tokens behind the cached ones of a page are not its own yet: they are left as they are
    first = torch.zeros(num, dtype=torch.long, device=x.device)
    first[s["table"].long()[torch.arange(at.numel(), device=x.device), at]] = p["old"] % ps
    keep = torch.arange(ps, device=x.device)[None, :] < first[:, None]
    again = (codes.view(torch.float8_e4m3fn).float() * _pow2((was - e).clamp(min=-126))[:, :, None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes.copy_(torch.where((grown[:, :, None] & keep[:, None, :])[..., None], again, codes))
    codes[page, :, slot] = (x.float() * _pow2(-e)[page][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    scales.copy_((e + 127).to(torch.uint8))


def _gather(s, codes, scales):
    """[seqs, max_len, heads, d]: the cached values of every sequence; zeros where it has no token."""
    p, ps = s["plan"], s["page"]
    j = torch.arange(p["max_len"], device=codes.device)
    page = s["table"].long()[:, j // ps].clamp(min=0)
    v = codes.view(torch.float8_e4m3fn).float()[page, :, (j % ps)[None, :].expand_as(page)]
    v = v * _pow2(scales.to(torch.int32) - 127)[page][..., None]
    return torch.where((j[None, :] < (p["old"] + p["new"])[:, None])[..., None, None], v, torch.zeros_like(v))


def _visible(s, pos):
    """Which keys a query at position pos sees."""
    j = torch.arange(s["plan"]["max_len"], device=pos.device)
    seen = j <= pos[..., None]
    return seen & (j > pos[..., None] - s["window"]) if s["window"] else seen


def _attend(s):
    p = s["plan"]
    rows, heads, d = s["q"].shape
    kvh = s["k_scales"].shape[1]
    seqs = p["old"].numel()
    k = _gather(s, s["k_codes"], s["k_scales"])
    v = _gather(s, s["v_codes"], s["v_scales"])
    q = torch.zeros(seqs, p["max_new"], heads, d, device=k.device)
    q[p["seq"], p["row"]] = s["q"].float()
    q = q.view(seqs, p["max_new"], kvh, heads // kvh, d).permute(0, 2, 3, 1, 4)                    # [seqs, kvh, group, new, d]
    sc = torch.matmul(q, k.permute(0, 2, 3, 1)[:, :, None]) / math.sqrt(d)
    pos = p["old"][:, None] + torch.arange(p["max_new"], device=k.device)
    sc = sc.masked_fill(~_visible(s, pos)[:, None, None], -math.inf)
    m = sc.amax(dim=-1, keepdim=True)
    sc = torch.exp(sc - m)
    l = sc.sum(dim=-1, keepdim=True)
    o = torch.matmul(sc, v.permute(0, 2, 1, 3)[:, :, None]) / l
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, p["max_new"], heads, d)[p["seq"], p["row"]].to(torch.bfloat16)
    lse = (m + torch.log(l))[..., 0].permute(0, 3, 1, 2).reshape(seqs, p["max_new"], heads)[p["seq"], p["row"]]
    return {"out": o, "lse": lse} if s["lse"] else {"out": o}


def run(s):
    op = s["op"]
    if op == "gemm":
        if own:
            from oxicuda_b200.blas import gemm_fp8_block128
            return gemm_fp8_block128(s["a"], s["w"], s["sa"], s["sw"], out_dtype=s["out"])
        return torch.matmul(_dense(s["a"], s["sa"], 1), _dense(s["w"], s["sw"], 128).t()).to(s["out"])
    if op == "norm":
        if own:
            from oxicuda_b200.kv_cache import rms_norm_quantize_fp8_block128
            got = rms_norm_quantize_fp8_block128(s["x"], s["gamma"], s["eps"], residual=s["residual"], want_y=s["y"])
            out = {"codes": got[0].view(torch.float8_e4m3fn), "scales": got[1]}
            if s["residual"] is not None:
                out["residual"] = s["residual"]
            if s["y"]:
                out["y"] = got[2]
            return out
        return _norm(s)
    if op == "swiglu":
        cols = s["gu"].shape[1] // 2
        if own:
            from oxicuda_b200.quant import swiglu_quantize_fp8_block128
            codes, scales = swiglu_quantize_fp8_block128(s["gu"][:, :cols], s["gu"][:, cols:])
            return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales}
        gate, up = s["gu"][:, :cols].float(), s["gu"][:, cols:].float()
        codes, scales = _quantize(gate * up / (1.0 + torch.exp(-gate)))
        return {"codes": codes, "scales": scales}
    if op == "append":
        if own:
            s["cache"].append(s["k"], s["v"], s["seq_lens"], s["table"], q_starts=s["starts"])
        else:
            _append_one(s, s["k_codes"], s["k_scales"], s["k"])
            _append_one(s, s["v_codes"], s["v_scales"], s["v"])
        return {"k": s["k_codes"].view(torch.float8_e4m3fn), "v": s["v_codes"].view(torch.float8_e4m3fn), "k_scales": s["k_scales"],
                "v_scales": s["v_scales"]}
    if own:
        got = s["cache"].attend(s["q"], s["seq_lens"], s["table"], q_starts=s["starts"], window=s["window"], want_lse=s["lse"])
        return {"out": got[0], "lse": got[1]} if s["lse"] else {"out": got}
    return _attend(s)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        kb = (k + 127) // 128
        return {"bytes": m * k + n * k + 4 * kb * (m + (n + 127) // 128) + m * n * (2 if case["out"] == "bf16" else 4), "flops": 2.0 * m * n * k}
    if op == "norm":
        e = case["rows"] * case["cols"]
        per = 2 + (4 if case["residual"] else 0) + 1 + (2 if case["y"] else 0)
        return {"bytes": e * per + 4 * case["rows"] * ((case["cols"] + 127) // 128) + 2 * case["cols"], "flops": 8.0 * e}
    if op == "swiglu":
        e = case["rows"] * case["cols"]
        return {"bytes": 5 * e + 4 * case["rows"] * ((case["cols"] + 127) // 128), "flops": 10.0 * e}
    # the mean sequence, as prepare() draws them: new tokens 0.8 of the figure where they are ragged, cached ones 0.75
    seqs, kvh, d = case["seqs"], case["kv_heads"], case["head_dim"]
    new = case["new"] if case["new"] <= 4 or seqs == 1 else 0.8 * case["new"] + 0.2 * case["new"] / seqs
    old = case["old"] if seqs == 1 else 0.75 * case["old"] + 0.25 * case["old"] / seqs
    if op == "append":
        return {"bytes": seqs * new * kvh * d * 2 * 3.0, "flops": seqs * new * kvh * d * 2 * 4.0}
    keys = old + new
    mean = old + (new + 1) / 2.0
    if case["window"]:
        mean, keys = min(mean, case["window"]), min(keys, case["window"] + new)
    return {"bytes": seqs * (keys * kvh * d * 2 + new * case["heads"] * d * 4.0), "flops": seqs * new * case["heads"] * d * 4.0 * mean}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _decode64():
    """The value of each E4M3 code."""
    t = torch.empty(256, dtype=torch.float64)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = math.ldexp(m / 8.0, -6) if e == 0 else math.ldexp(1.0 + m / 8.0, e - 7)
        t[c] = float("nan") if (c & 127) == 127 else (-v if c & 128 else v)
    return t.cuda()


def _encode64(x):
    """The E4M3 value nearest to x, ties to the even one, at most 448 in size."""
    a = x.abs().clamp(max=E4M3_MAX)
    step = torch.ldexp(torch.ones_like(a), torch.frexp(a)[1].clamp(min=-5) - 4)     # 2^(exponent - 3), and 2^-9 below 2^-6
    return torch.copysign(torch.round(a / step) * step, x)


def _block64(y):
    rows, cols = y.shape
    nb = (cols + 127) // 128
    s = torch.ones(rows, nb, dtype=torch.float64, device=y.device)
    for b in range(nb):
        top = y[:, 128 * b: 128 * b + 128].abs().max(dim=1).values
        s[:, b] = torch.where(top > 0, top / E4M3_MAX, s[:, b])
    return _encode64(y / s[:, torch.arange(cols, device=y.device) // 128]), s


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    lut = _decode64()
    if op == "gemm":
        kb = st["sa"].shape[1]
        out = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
        col = torch.arange(case["n"], device="cuda") // 128
        for b in range(kb):
            part = lut[st["a"][:, 128 * b: 128 * b + 128].long()] @ lut[st["w"][:, 128 * b: 128 * b + 128].long()].t()
            out += part * st["sa"][:, b, None].double() * st["sw"][col, b].double()
        return out
    if op == "norm":
        x = st["x"].double()
        out = {}
        if st["residual"] is not None:
            x = (x + st["residual"].double()).float().to(torch.bfloat16).double()
            out["residual"] = x
        y = x * torch.rsqrt(x.square().sum(dim=1, keepdim=True) / case["cols"] + st["eps"]) * st["gamma"].double()
        out["codes"], out["scales"] = _block64(y)
        if case["y"]:
            out["y"] = y
        return out
    if op == "swiglu":
        gate, up = st["gu"].double().chunk(2, dim=1)
        codes, scales = _block64(gate * torch.sigmoid(gate) * up)
        return {"codes": codes, "scales": scales}
    ps, table, lens = case["page"], st["table"].tolist(), st["seq_lens"].tolist()
    starts = list(range(case["seqs"] + 1)) if st["starts"] is None else st["starts"].tolist()
    if op == "append":
        if case["seqs"] * case["new"] * case["kv_heads"] > 80000:      # a page at a time takes too long beyond that
            return None
        out = {}
        for name in ("k", "v"):
            val, sc = lut[st[name + "_codes"].long()], st[name + "_scales"].long() - 127
            for b, n in enumerate(lens):
                first = n - (starts[b + 1] - starts[b])
                for i in range(first // ps, (n - 1) // ps + 1):
                    pg, lo, hi = table[b][i], max(first, i * ps), min(n, (i + 1) * ps)
                    x = st[name][starts[b] + lo - first: starts[b] + hi - first].double()
                    # (the inputs have 8 significant bits: a margin of 1e-9 takes nothing from a power of two but log2's own error)
                    e = torch.ceil(torch.log2(x.abs().amax(dim=(0, 2)).clamp(min=1e-30) / E4M3_MAX) - 1e-9).long().clamp(MIN_EXP, MAX_EXP)
                    if lo > i * ps:
                        e = torch.maximum(e, sc[pg])
                        val[pg, :, : lo - i * ps] = _encode64(val[pg, :, : lo - i * ps] * torch.exp2((sc[pg] - e).double())[:, None, None])
                    sc[pg] = e
                    val[pg, :, lo - i * ps: hi - i * ps] = _encode64(x.transpose(0, 1) * torch.exp2(-e.double())[:, None, None])
            out[name], out[name + "_scales"] = val, None
        return out
    kvh, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["q"].shape[:2], dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        j = torch.arange(n, device="cuda")
        pg = st["table"][b].long()[j // ps]
        pos = n - (r1 - r0) + torch.arange(r1 - r0, device="cuda")
        hide = j[None, :] > pos[:, None]
        if case["window"]:
            hide = hide | (j[None, :] <= pos[:, None] - case["window"])
        for h in range(kvh):
            k = lut[st["k_codes"][pg, h, j % ps].long()] * torch.exp2(st["k_scales"][pg, h].double() - 127.0)[:, None]
            v = lut[st["v_codes"][pg, h, j % ps].long()] * torch.exp2(st["v_scales"][pg, h].double() - 127.0)[:, None]
            q = st["q"][r0:r1, h * group: (h + 1) * group].double()
            w = torch.einsum("qgd,kd->gqk", q, k).div_(math.sqrt(case["head_dim"])).masked_fill_(hide[None], -math.inf)
            lse[r0:r1, h * group: (h + 1) * group] = torch.logsumexp(w, dim=2).t()
            out[r0:r1, h * group: (h + 1) * group] = torch.einsum("gqk,kd->qgd", torch.softmax(w, dim=2), v)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
