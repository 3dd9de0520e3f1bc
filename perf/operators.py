"""Operators of the 8-bit paged K/V cache: quantising append, dequantising read,
decode and chunked-prefill attention over the 8-bit pages, and page copies.

The cache holds e4m3 codes ``[L, P, Hkv, bs, D]`` and one fp32 scale per
(layer, block, KV head), a power of two; a value is ``code * scale``.  ``run``
is one pass through an operator: its plain form in elementary torch
operations, or (``own``) the call a user makes of ``barellm_b200.ops``.
"""

import math

import numpy as np
import torch

own = False

F8 = torch.float8_e4m3fn
F8_MAX = 448.0
MIN_EXP, MAX_EXP = -100, 119  # range of the scales' exponents
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    c = []
    # One decode step of a small batch (Qwen3-0.6B heads): one token per row into a half-filled block.
    c.append(dict(name="append_step_b4", op="append", dtype="bf16", batch=4, hq=16, hkv=8, dim=128, bs=16, layers=2,
                  lo=100, hi=700, new_lo=1, new_hi=1, lens_seed=1))
    # One decode step of a full batch (Qwen3-8B heads).
    c.append(dict(name="append_step_b256", op="append", dtype="bf16", batch=256, hq=32, hkv=8, dim=128, bs=16, layers=2,
                  lo=200, hi=2000, new_lo=1, new_hi=1, lens_seed=2))
    # Packed prompt chunks of 32 requests, starting anywhere in a block.
    c.append(dict(name="append_chunks", op="append", dtype="bf16", batch=32, hq=32, hkv=8, dim=128, bs=16, layers=1,
                  lo=0, hi=4000, new_lo=512, new_hi=2048, lens_seed=3))
    # Dense read of a batch's cache (Qwen3-0.6B heads), zero padded.
    c.append(dict(name="gather_b3", op="gather", dtype="f16", batch=3, hq=16, hkv=8, dim=128, bs=16, layers=2,
                  lo=33, hi=500, lens_seed=4))
    c.append(dict(name="gather_b64", op="gather", dtype="bf16", batch=64, hq=16, hkv=8, dim=128, bs=16, layers=1,
                  lo=128, hi=4096, lens_seed=5))
    # Decode: a single short request, where latency counts.
    c.append(dict(name="decode_b1_short", op="decode", dtype="bf16", batch=1, hq=16, hkv=8, dim=128, bs=16, layers=2,
                  lo=777, hi=777, lens_seed=6))
    # Decode: an ordinary serving batch (Qwen3-0.6B heads).
    c.append(dict(name="decode_b64", op="decode", dtype="f16", batch=64, hq=16, hkv=8, dim=128, bs=16, layers=1,
                  lo=128, hi=4096, lens_seed=7))
    # Decode: long contexts (Qwen3-8B heads).
    c.append(dict(name="decode_b64_long", op="decode", dtype="bf16", batch=64, hq=32, hkv=8, dim=128, bs=16, layers=1,
                  lo=1024, hi=32768, lens_seed=8))
    # Prefill: a few odd chunks over short prefixes.
    c.append(dict(name="prefill_b3", op="prefill", dtype="f16", batch=3, hq=16, hkv=8, dim=128, bs=16, layers=2,
                  lo=0, hi=600, new_lo=17, new_hi=130, lens_seed=9))
    # Prefill: prompt chunks over cached prefixes (Qwen3-8B heads).
    c.append(dict(name="prefill_b8", op="prefill", dtype="bf16", batch=8, hq=32, hkv=8, dim=128, bs=16, layers=1,
                  lo=0, hi=8192, new_lo=512, new_hi=1024, lens_seed=10))
    # Page copies: the last pages of 8 forked requests, all 28 layers, 8-bit pages with their scales.
    c.append(dict(name="copy_fork8_fp8", op="copy", dtype="fp8", pairs=8, hkv=8, dim=128, bs=16, layers=28, spare=120))
    # Page copies: compaction of a bf16 pool, all 28 layers.
    c.append(dict(name="copy_compact_bf16", op="copy", dtype="bf16", pairs=1024, hkv=8, dim=128, bs=16, layers=28,
                  spare=64))
    return c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "gather", "decode", "decode", "prefill", "copy"])
    hq, hkv = rng.choice([(16, 8)] * 4 + [(32, 8)] * 4 + [(8, 8), (16, 1), (12, 4), (40, 8)])
    dim = rng.choice([128] * 9 + [64, 256, 80])
    bs = rng.choice([16] * 9 + [32, 8])
    if op == "copy":
        c = dict(op=op, dtype=rng.choice(["fp8", "fp8", "bf16", "f32"]), pairs=_log(rng, 1, 1000), hkv=hkv, dim=dim, bs=bs,
                 layers=rng.choice([1, 5, 28, 36]), spare=rng.randint(0, 200))
    else:
        c = dict(op=op, dtype=rng.choice(["bf16"] * 5 + ["f16"] * 3 + ["f32"]), batch=_log(rng, 1, 256), hq=hq,
                 hkv=hkv, dim=dim, bs=bs, layers=rng.choice([1, 2, 3]), lens_seed=rng.randint(0, 1 << 30))
        c["hi"] = _log(rng, 1, {"append": 4000, "gather": 4096, "decode": 32768, "prefill": 8192}[op])
        c["lo"] = rng.randint(1 if op in ("gather", "decode") else 0, max(1, c["hi"] // 2))
        if op == "append":
            c["new_hi"] = rng.choice([1, _log(rng, 1, 2048)])
            c["new_lo"] = rng.randint(1, c["new_hi"])
        if op == "prefill":
            c["batch"] = min(c["batch"], 16)
            c["new_hi"] = _log(rng, 2, 1024)
            c["new_lo"] = rng.randint(1, c["new_hi"])
    # no dearer than the largest listed case of the same operator, nor as dense a padded plain form
    most = [work(x) for x in listed() if x["op"] == op]
    key = "pairs" if op == "copy" else "batch"
    while c[key] > 1 and (work(c)["bytes"] > max(w["bytes"] for w in most)
                          or work(c)["flops"] > max(w["flops"] for w in most) or _padded(c) > 2.2e9):
        c[key] = (c[key] + 1) // 2
    return c


def _lens(case):
    """(cached lengths before the call, new tokens) per row, from the case alone."""
    r = np.random.RandomState(case["lens_seed"])
    lens = r.randint(case["lo"], max(case["lo"], case["hi"]) + 1, case["batch"])
    new = r.randint(case.get("new_lo", 0), case.get("new_hi", 0) + 1, case["batch"])
    return lens.astype(np.int64), new.astype(np.int64)


def _padded(case):
    """Elements of the largest tensor of the plain form."""
    if case["op"] == "copy":
        return 0
    lens, new = _lens(case)
    t = int((lens + new).max())
    if case["op"] == "prefill":
        return case["batch"] * case["hq"] * int(new.max()) * t
    if case["op"] == "append":
        return case["batch"] * case["hkv"] * (int(new.max()) + 2 * case["bs"]) * case["dim"]
    return case["batch"] * case["hkv"] * t * case["dim"]


def work(case):
    hkv, d, bs = case["hkv"], case["dim"], case["bs"]
    if case["op"] == "copy":
        es = 1 if case["dtype"] == "fp8" else ES[case["dtype"]]
        page = hkv * bs * d * es + (4 * hkv if case["dtype"] == "fp8" else 0)
        return {"bytes": 2 * 2 * case["pairs"] * case["layers"] * page, "flops": 0}
    es = ES[case["dtype"]]
    lens, new = _lens(case)
    if case["op"] == "append":
        n = int(new.sum())
        blocks = int(((lens + new + bs - 1) // bs - lens // bs).sum())
        return {"bytes": 2 * n * hkv * d * (es + 1) + 2 * blocks * hkv * 4, "flops": 0}
    total = lens + new
    n = int(total.sum())
    codes = 2 * n * hkv * d + 2 * int(((total + bs - 1) // bs).sum()) * hkv * 4
    if case["op"] == "gather":
        return {"bytes": codes + 2 * case["batch"] * int(total.max()) * hkv * d * es, "flops": 0}
    hq = case["hq"]
    if case["op"] == "decode":
        return {"bytes": codes + 2 * case["batch"] * hq * d * es, "flops": 4 * hq * d * n}
    seen = int((new * lens + new * (new + 1) // 2).sum())
    return {"bytes": codes + 2 * int(new.sum()) * hq * d * es, "flops": 4 * hq * d * seen}


# --- inputs ----------------------------------------------------------------


def _pow2_scale(amax):
    """Smallest 2^k with amax <= 448 * 2^k, k in [MIN_EXP, MAX_EXP] (fp32)."""
    m, e = torch.frexp(amax)
    k = torch.where(m <= 0.875, e - 9, e - 8).clamp(MIN_EXP, MAX_EXP)
    k = torch.where(amax > 0, k, torch.full_like(k, MIN_EXP))
    return torch.ldexp(torch.ones_like(amax), k)


def _encode(x, scale):
    """e4m3 codes of x / scale (round to nearest even, saturating)."""
    return (x / scale).clamp(-F8_MAX, F8_MAX).to(F8)


def _pool(g, layers, blocks, hkv, bs, d, spread):
    """An 8-bit pool filled as a cache is: token magnitudes vary, a few channels are much larger than the rest."""
    dev = torch.device("cuda")
    codes = torch.empty((layers, blocks, hkv, bs, d), dtype=F8, device=dev)
    scales = torch.empty((layers, blocks, hkv), dtype=torch.float32, device=dev)
    gain = torch.exp(spread * torch.randn((hkv, 1, d), generator=g, device=dev))
    step = max(1, (1 << 28) // (hkv * bs * d))
    for l in range(layers):
        for i in range(0, blocks, step):
            n = min(step, blocks - i)
            x = torch.randn((n, hkv, bs, d), generator=g, device=dev) * gain
            s = _pow2_scale(x.abs().amax(dim=(2, 3)))
            scales[l, i:i + n] = s
            codes[l, i:i + n] = _encode(x, s[..., None, None])
    return codes, scales, gain


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    hkv, d, bs, layers = case["hkv"], case["dim"], case["bs"], case["layers"]
    s = dict(op=case["op"], bs=bs, layer=layers - 1)
    if case["op"] == "copy":
        n = case["pairs"]
        blocks = 2 * n + case["spare"]
        ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))[: 2 * n].tolist()
        s["src"], s["dst"] = ids[:n], ids[n:]
        shape = (layers, blocks, hkv, bs, d)
        if case["dtype"] == "fp8":
            s["kc"], s["ks"], _ = _pool(g, layers, blocks, hkv, bs, d, 0.5)
            s["vc"], s["vs"], _ = _pool(g, layers, blocks, hkv, bs, d, 0.2)
        else:
            s["kc"] = torch.randn(shape, generator=g, device=dev, dtype=DTYPES[case["dtype"]])
            s["vc"] = torch.randn(shape, generator=g, device=dev, dtype=DTYPES[case["dtype"]])
            s["ks"] = s["vs"] = None
        return s
    dt = DTYPES[case["dtype"]]
    s["dtype"] = dt
    lens, new = _lens(case)
    total = lens + new
    nb = -(-total // bs)
    blocks = int(nb.sum()) + 7
    width = int(nb.max())
    ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).numpy()
    bt = np.full((case["batch"], width), -1, dtype=np.int32)
    at = 0
    for b in range(case["batch"]):
        bt[b, : nb[b]] = ids[at : at + nb[b]]
        at += nb[b]
    s["bt"] = torch.from_numpy(bt).to(dev)
    s["kc"], s["ks"], kgain = _pool(g, layers, blocks, hkv, bs, d, 0.5)
    s["vc"], s["vs"], _ = _pool(g, layers, blocks, hkv, bs, d, 0.2)
    s["start"] = torch.from_numpy(lens.astype(np.int32)).to(dev)
    s["lens"] = torch.from_numpy(total.astype(np.int32)).to(dev)
    s["max_len"] = int(total.max())
    s["total_blocks"] = int(nb.sum())
    if case["op"] in ("append", "prefill"):
        off = np.zeros(case["batch"] + 1, dtype=np.int32)
        off[1:] = np.cumsum(new)
        s["off"] = torch.from_numpy(off).to(dev)
        s["max_new"] = int(new.max())
        n = int(new.sum())
    if case["op"] == "append":
        # packed tokens as the projections leave them: [1, H, N, D] over [N, H, D] memory
        s["k"] = (torch.randn((n, hkv, d), generator=g, device=dev) * kgain[:, 0]).to(dt).unsqueeze(0).transpose(1, 2)
        s["v"] = torch.randn((n, hkv, d), generator=g, device=dev).to(dt).unsqueeze(0).transpose(1, 2)
    if case["op"] == "decode":
        s["q"] = torch.randn((case["batch"], case["hq"], d), generator=g, device=dev).to(dt)
    if case["op"] == "prefill":
        s["q"] = torch.randn((n, case["hq"], d), generator=g, device=dev).to(dt).unsqueeze(0).transpose(1, 2)
    return s


# --- plain forms -------------------------------------------------------------


def _pages(pool, bt):
    """pool[bt] for 8-bit pools, -1 entries read block 0 (masked by the caller)."""
    return pool.view(torch.uint8)[bt.clamp(min=0).long()].view(F8)


def _dense(s, pool, scale):
    """fp32 values of a layer's cached tokens, [B, Hkv, W * bs, D], zeros behind each length."""
    bt, bs, l = s["bt"], s["bs"], s["layer"]
    x = _pages(pool[l], bt).float() * scale[l][bt.clamp(min=0).long()][..., None, None]
    b, w, h, _, d = x.shape
    x = x.transpose(1, 2).reshape(b, h, w * bs, d)
    live = torch.arange(w * bs, device=x.device)[None, :] < s["lens"][:, None]
    return torch.where(live[:, None, :, None], x, 0.0)


def _softmax_pv(score, seen, v):
    """softmax over the seen keys times v, fp32; a row that sees nothing gives zeros."""
    score = torch.where(seen, score, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, 0.0))
    den = p.sum(dim=-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(den > 0, den, 1.0)


def _append_half(s, pool, scales, x):
    """Plain append of packed tokens x [N, Hkv, D] into one layer's codes and scales."""
    bt, bs = s["bt"], s["bs"]
    start, off = s["start"].long(), s["off"].long()
    n_new = off[1:] - off[:-1]
    touched = (s["max_new"] + bs - 1) // bs + 1
    lb = start[:, None] // bs + torch.arange(touched, device=x.device)  # [B, n] logical blocks
    pos = lb[..., None] * bs + torch.arange(bs, device=x.device)  # [B, n, bs]
    is_new = (pos >= start[:, None, None]) & (pos < (start + n_new)[:, None, None])
    is_old = pos < start[:, None, None]
    use = is_new.any(dim=-1)  # blocks that receive a token
    lb, is_new, is_old = lb[use], is_new[use], is_old[use]
    row = torch.arange(bt.shape[0], device=x.device)[:, None].expand_as(use)[use]
    phys = bt[row, lb].long()
    tok = (off[:-1][row][:, None] + pos[use] - start[row][:, None]).clamp(0, x.shape[0] - 1)
    xs = torch.where(is_new[..., None, None], x[tok].float(), 0.0).transpose(1, 2)  # [M, Hkv, bs, D]
    amax = torch.where(torch.isfinite(xs), xs.abs(), 0.0).amax(dim=(2, 3))
    old_scale = torch.where(is_old.any(dim=-1)[:, None], scales[phys], 0.0)
    new_scale = torch.maximum(_pow2_scale(amax), old_scale)
    old = _pages(pool, phys)
    moved = _encode(old.float() * old_scale[..., None, None], new_scale[..., None, None])
    fresh = _encode(xs, new_scale[..., None, None])
    codes = torch.where(is_new[:, None, :, None], fresh.view(torch.uint8),
                        torch.where(is_old[:, None, :, None], moved.view(torch.uint8), old.view(torch.uint8)))
    pool.view(torch.uint8)[phys] = codes
    scales[phys] = new_scale


def _run_plain(s):
    op, l = s["op"], s.get("layer")
    if op == "copy":
        src = torch.tensor(s["src"], device=s["kc"].device)
        dst = torch.tensor(s["dst"], device=s["kc"].device)
        kc, vc = s["kc"], s["vc"]
        if s["ks"] is not None:
            kc, vc = kc.view(torch.uint8), vc.view(torch.uint8)
            s["ks"][:, dst] = s["ks"][:, src]
            s["vs"][:, dst] = s["vs"][:, src]
        kc[:, dst] = kc[:, src]
        vc[:, dst] = vc[:, src]
        return _copied(s)
    if op == "append":
        _append_half(s, s["kc"][l], s["ks"][l], s["k"][0].transpose(0, 1))
        _append_half(s, s["vc"][l], s["vs"][l], s["v"][0].transpose(0, 1))
        return s["kc"], s["vc"], s["ks"], s["vs"]
    dt = s["dtype"]
    if op == "gather":
        k = _dense(s, s["kc"], s["ks"])[:, :, : s["max_len"]]
        v = _dense(s, s["vc"], s["vs"])[:, :, : s["max_len"]]
        top = torch.finfo(dt).max
        return k.clamp(-top, top).to(dt).contiguous(), v.clamp(-top, top).to(dt).contiguous()
    k = _dense(s, s["kc"], s["ks"])
    b, h, t, d = k.shape
    keys = torch.arange(t, device=k.device)
    if op == "decode":
        q = s["q"].float().view(b, h, -1, d)
        score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(d)
        del k
        seen = (keys[None, :] < s["lens"][:, None])[:, None, None, :]
        out = _softmax_pv(score, seen, _dense(s, s["vc"], s["vs"]))
        return out.reshape(b, -1, d).to(dt)
    # prefill: queries padded to [B, C]
    q = s["q"][0].transpose(0, 1).float()  # [N, Hq, D]
    off = s["off"].long()
    c = torch.arange(s["max_new"], device=q.device)
    n_new = off[1:] - off[:-1]
    live = c[None, :] < n_new[:, None]
    tok = (off[:-1, None] + c).clamp(max=q.shape[0] - 1)
    qp = q[tok].view(b, s["max_new"], h, -1, d).permute(0, 2, 3, 1, 4)  # [B, Hkv, G, C, D]
    score = torch.matmul(qp.reshape(b, h, -1, d), k.transpose(2, 3)) / math.sqrt(d)
    del k
    last = s["lens"].long()[:, None] - n_new[:, None] + c  # the last key that query c sees
    seen = (keys[None, None, :] <= last[:, :, None])[:, None, None].expand(b, h, qp.shape[2], -1, t)
    out = _softmax_pv(score, seen.reshape(b, h, -1, t), _dense(s, s["vc"], s["vs"]))
    out = out.view(b, h, qp.shape[2], -1, d).permute(0, 3, 1, 2, 4).reshape(b, s["max_new"], -1, d)
    return out[live].to(dt).unsqueeze(0).transpose(1, 2)


def _copied(s):
    return [t for t in (s["kc"], s["vc"], s["ks"], s["vs"]) if t is not None]


# --- the framework's calls -----------------------------------------------------


def _run_own(s):
    from barellm_b200 import ops

    op = s["op"]
    if op == "copy":
        ops.copy_blocks(s["kc"], s["vc"], s["src"], s["dst"], key_scale=s["ks"], value_scale=s["vs"])
        return _copied(s)
    cache = (s["kc"], s["vc"], s["ks"], s["vs"], s["layer"], s["bt"])
    if op == "append":
        ops.paged_append_fp8(*cache, s["start"], s["k"], s["v"], new_offsets=s["off"], max_new_tokens=s["max_new"])
        return s["kc"], s["vc"], s["ks"], s["vs"]
    if op == "gather":
        return ops.paged_gather_fp8(*cache, s["lens"], s["max_len"], dtype=s["dtype"])
    if op == "decode":
        return ops.paged_decode_fp8(s["q"], *cache, s["lens"], s["max_len"])
    return ops.paged_prefill_fp8(s["q"], *cache, s["lens"], s["max_len"], total_blocks=s["total_blocks"],
                                 q_offsets=s["off"], max_q_len=s["max_new"])


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# --- definition in 64 bits -------------------------------------------------------


def _e4m3_round(x):
    """The nearest e4m3 value of x (float64), ties to even mantissa, saturating at 448; NaN stays."""
    a = x.abs().clamp(max=F8_MAX)
    e = torch.floor(torch.log2(torch.where(a > 0, a, 1.0))).clamp(min=-6)
    e = torch.where(a >= torch.exp2(e + 1), e + 1, e)
    e = torch.where((a < torch.exp2(e)) & (e > -6), e - 1, e)
    ulp = torch.exp2(e - 3)
    return torch.copysign(torch.round(a / ulp) * ulp, x)


def _row64(s, pool, scales, b):
    """One row's cached tokens in float64, [Hkv, len, D]."""
    n = int(s["lens"][b])
    ids = s["bt"][b, : -(-n // s["bs"])].long()
    l = s["layer"]
    x = pool[l].view(torch.uint8)[ids].view(F8).double() * scales[l][ids].double()[:, :, None, None]
    h, d = x.shape[1], x.shape[3]
    return x.permute(1, 0, 2, 3).reshape(h, -1, d)[:, :n]


def _scale64(amax):
    k = MIN_EXP
    while k < MAX_EXP and amax > F8_MAX * 2.0 ** k:
        k += 1
    return 2.0 ** k


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        for t in _copied(s):
            raw = t.view(torch.uint8) if t.dtype == F8 else t
            for a, b in zip(s["src"], s["dst"]):
                raw[:, b].copy_(raw[:, a])
        return [t if t.dtype == torch.float32 else t.float() for t in _copied(s)] if s["kc"].numel() < 1 << 28 else None
    rows = case["batch"]
    if case["op"] == "append":
        off = s["off"].tolist()
        if off[-1] > 20000:
            return None
        out = []
        for pool, scales, x in ((s["kc"], s["ks"], s["k"]), (s["vc"], s["vs"], s["v"])):
            l, bs = s["layer"], s["bs"]
            vals, sc = pool.double(), scales.double()
            for b in range(rows):
                start, new = int(s["start"][b]), x[0, :, off[b]:off[b + 1]].double()
                end = start + new.shape[1]
                for j in range(start // bs, -(-end // bs)):
                    p0, p1 = max(start, j * bs), min(end, (j + 1) * bs)
                    page, part = vals[l, int(s["bt"][b, j])], new[:, p0 - start:p1 - start]
                    sp = sc[l, int(s["bt"][b, j])]
                    need = torch.tensor([_scale64(float(a)) for a in part.abs().amax(dim=(1, 2))], dtype=torch.float64,
                                        device=x.device)
                    kept = p0 - j * bs
                    use = torch.maximum(need, sp) if kept else need
                    page[:, :kept] = _e4m3_round(page[:, :kept] * (sp / use)[:, None, None])
                    page[:, kept:p1 - j * bs] = _e4m3_round(part / use[:, None, None])
                    sp.copy_(use)
            out.append((vals, sc))
        return out[0][0], out[1][0], out[0][1], out[1][1]
    if case["op"] == "gather":
        top = torch.finfo(s["dtype"]).max
        out = []
        for pool, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
            o = torch.zeros((rows, case["hkv"], s["max_len"], case["dim"]), dtype=torch.float64, device=pool.device)
            for b in range(rows):
                x = _row64(s, pool, scales, b)
                o[b, :, : x.shape[1]] = x.clamp(-top, top)
            out.append(o)
        return tuple(out)
    hq, d, g = case["hq"], case["dim"], case["hq"] // case["hkv"]
    outs = []
    for b in range(rows):
        k, v = _row64(s, s["kc"], s["ks"], b), _row64(s, s["vc"], s["vs"], b)
        n = k.shape[1]
        if case["op"] == "decode":
            q = s["q"][b].double()[:, None]
        else:
            q = s["q"][0, :, int(s["off"][b]):int(s["off"][b + 1])].double()
        c = q.shape[1]
        o = torch.zeros((hq, c, d), dtype=torch.float64, device=q.device)
        for h in range(hq):
            for i in range(0, c, 256):
                z = q[h, i:i + 256] @ k[h // g].T / math.sqrt(d)
                m = torch.arange(n, device=q.device)[None] > (n - c + i + torch.arange(z.shape[0], device=q.device))[:, None]
                o[h, i:i + 256] = torch.softmax(z.masked_fill(m, -math.inf), dim=-1) @ v[h // g]
        outs.append(o)
    if case["op"] == "decode":
        return torch.stack([o[:, 0] for o in outs])
    return torch.cat(outs, dim=1).unsqueeze(0)
