"""Performance cases of the 4-bit KV cache: the rows of a layer on their way into it, the
cache itself, and the attention over it.

  rope       norms of queries and keys for each head with the position rotation in the same
             pass (qk_norm_rope), one position axis or several, on slices of a fused projection
  rope_kv    the same with the keys and values written to the 4-bit cache (norm_rope_append)
  cache      rows quantised into the cache and read back as values (KVCache.append, .read)
  attention  the schedule of a step and the paged attention of its rows over the cache
             (attention_plan, attention); one row a sequence is plain decoding
  layer      a whole layer of a step: norm and rotation, plan, draft rows appended and attended,
             and the appended rows read back

The cache holds, for each token and kv head and for keys and values apart, codes n in 0..15 with
a scale s and a zero point z: lo = min(0, x), hi = max(0, x), s = (hi - lo) / 15 rounded up to five
significant bits, z = rint(-lo / s), n = rint(x / s) + z kept in 0..15. It stands for s (n - z).

The context lengths of a case follow from the case alone, so its work is a fixed number; block
placement and all values come from the seed.
"""
import math
import zlib

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 16
EPS = 1e-6


def rope(tokens, q_heads, kv_heads, dim, io, axes=1, pairs=False, rotary=0, far=0):
    return {"kind": "rope", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "io": io,
            "axes": axes, "pairs": pairs, "rotary": rotary or dim, "far": far}


def rope_kv(tokens, q_heads, kv_heads, dim, io, far=0):
    return {"kind": "rope_kv", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "io": io,
            "axes": 1, "pairs": False, "rotary": dim, "far": far}


def cache(tokens, kv_heads, dim, io, first=0):
    return {"kind": "cache", "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "io": io, "first": first}


def attention(seqs, rows, q_heads, kv_heads, dim, lo, hi, io="bf16", ragged=False, kind="attention"):
    return {"kind": kind, "seqs": seqs, "rows": rows, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "ctx_lo": lo, "ctx_hi": hi, "io": io, "ragged": ragged}


def listed():
    named = {
        # One user chatting: the five rows of one verify step, nothing but a launch.
        "rope-single": rope(5, 32, 8, 128, "bf16", far=3001),
        # A long prompt of a vision-language model: time, height and width positions.
        "rope-prompt-axes": rope(32768, 32, 8, 128, "bf16", axes=3),
        # The verify rows of 64 sequences in one layer: rotated, their keys and values quantised.
        "rope-kv-8b": rope_kv(384, 32, 8, 128, "bf16", far=8192),
        # A prompt's chunk straight into the cache.
        "rope-kv-prompt": rope_kv(8192, 32, 8, 128, "bf16"),
        # The draft rows of one sequence, ending inside a block.
        "cache-step": cache(5, 8, 128, "bf16", first=3001),
        # A long prompt's keys and values written, and read back for another kernel's use.
        "cache-prompt": cache(32768, 8, 128, "bf16"),
        # One user chatting: a single sequence.
        "attn-single": attention(1, 5, 32, 8, 128, 3001, 3001),
        # Plain decoding (one row a sequence) in a large batch.
        "attn-decode": attention(128, 1, 32, 8, 128, 256, 2048),
        # The 8B shape's verify step: 64 sequences, five drafts.
        "attn-8b": attention(64, 6, 32, 8, 128, 1024, 8192),
        # Long documents: 8 sequences of 16k to 32k keys, eight drafts.
        "attn-long": attention(8, 9, 32, 8, 128, 16384, 32768),
        # Head_dim 64, drafts of uneven length.
        "attn-dim64": attention(16, 5, 32, 8, 64, 512, 4096, io="f16", ragged=True),
        # A whole layer of the 3B shape's step.
        "layer-3b": attention(32, 5, 24, 8, 128, 512, 4096, kind="layer"),
    }
    return [dict(c, name=n) for n, c in named.items()]


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    kind = rng.choice(["rope", "rope_kv", "cache", "attention", "attention", "layer"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    dim = rng.choice([64, 128, 128])
    io = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "rope":
        return rope(spread(1, 16384), q_heads, kv_heads, rng.choice([64, 80, 128, 256]), io, axes=rng.randint(1, 4),
                    pairs=rng.random() < 0.3, rotary=rng.choice([0, 32, 64]), far=rng.choice([0, 5000, 1000000]))
    if kind == "rope_kv":
        return rope_kv(spread(1, 6000), q_heads, kv_heads, dim, rng.choice(["bf16", "f16"]), far=rng.choice([0, 5000, 200000]))
    if kind == "cache":
        return cache(spread(1, 32768), kv_heads, dim, io, first=rng.randint(0, 5000))
    seqs = spread(1, 96)
    rows = rng.randint(1, 9)
    most = max(2400, min(300000, 50000000 // (rows * q_heads)))
    hi = max(24, min(32768, spread(24, most) // seqs + rng.randint(0, 15)))
    lo = max(1, hi // rng.choice([1, 2, 8]))
    return attention(seqs, rows, q_heads, kv_heads, dim, lo, hi, io=io, ragged=rng.random() < 0.4, kind=kind)


# ---- the shape of a case, fixed by the case alone ----

def lengths(case):
    """Cached tokens before the step's rows and rows of each sequence."""
    key = "|".join("%s=%s" % kv for kv in sorted(case.items()) if kv[0] != "name")
    r = np.random.RandomState(zlib.crc32(key.encode()) & 0x7fffffff)
    ctx = r.randint(case["ctx_lo"], case["ctx_hi"] + 1, case["seqs"])
    rows = r.randint(1, case["rows"] + 1, case["seqs"]) if case["ragged"] else np.full(case["seqs"], case["rows"])
    return ctx, rows


def work(case):
    dim, io = case["dim"], BYTES[case["io"]]
    if case["kind"] in ("rope", "rope_kv"):
        n, hq, hk = case["tokens"], case["q_heads"], case["kv_heads"]
        moved = 2 * n * (hq + hk) * dim * io
        if case["kind"] == "rope_kv":  # q once in and out, k and v in, the cache's bytes, read back in `io`
            moved = 2 * n * hq * dim * io + 2 * n * hk * dim * io + 2 * n * hk * (dim + 4) + 2 * n * hk * dim * io
        return {"bytes": moved, "flops": 10 * n * (hq + hk) * dim}
    if case["kind"] == "cache":
        n, hk = case["tokens"], case["kv_heads"]
        return {"bytes": 4 * n * hk * dim * io + 2 * n * hk * (dim + 4), "flops": 12 * n * hk * dim}
    ctx, rows = lengths(case)
    keys = int((ctx + rows).sum())
    nrow = int(rows.sum())
    moved = keys * case["kv_heads"] * (dim + 4) + 2 * nrow * case["q_heads"] * dim * io
    flops = int((4 * dim * case["q_heads"] * rows * (ctx + rows)).sum())
    if case["kind"] == "layer":
        moved += nrow * dim * io * (2 * case["q_heads"] + 6 * case["kv_heads"])
        flops += 10 * nrow * (case["q_heads"] + case["kv_heads"]) * dim
    return {"bytes": moved, "flops": flops}


# ---- inputs ----

def generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def frequencies(case):
    n = case.get("rotary", case["dim"]) // 2
    return torch.tensor(10000.0 ** (-np.arange(n) / n), dtype=torch.float32, device="cuda")


def axis_of_pair(case):
    """Pair j of the rotation turns by the positions of this axis: sections of near equal length."""
    axes, n = case.get("axes", 1), case.get("rotary", case["dim"]) // 2
    return [min(axes - 1, j * axes // n) for j in range(n)]


def projected(case, g, n):
    """The fused projection's rows [n, (q heads + 2 kv heads) * dim] (a few channels of the keys
    larger, as models have them), the norms' weights and the positions' frequencies."""
    hq, hk, dim, io = case["q_heads"], case["kv_heads"], case["dim"], TORCH[case["io"]]
    x = normal(g, n, hq + 2 * hk, dim) * (0.5 + torch.rand(n, 1, 1, generator=g, device="cuda"))
    x[:, hq:hq + hk, :: max(1, dim // 4)] *= 4.0
    return {"qkv": x.to(io).reshape(n, (hq + 2 * hk) * dim), "freq": frequencies(case),
            "q_weight": (1.0 + 0.2 * normal(g, dim)).to(io), "k_weight": (1.0 + 0.2 * normal(g, dim)).to(io)}


def split(case, qkv):
    hq, hk, dim = case["q_heads"], case["kv_heads"], case["dim"]
    x = qkv.view(qkv.shape[0], hq + 2 * hk, dim)
    return x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]


def blocks_for(g, counts):
    """Block tables [sequences, most blocks] over a shuffled pool, and the pool's block count."""
    most, total = int(max(counts)), int(sum(counts))
    tables = np.zeros((len(counts), most), np.int64)
    at = np.concatenate([[0], np.cumsum(counts)])
    for b, c in enumerate(counts):
        tables[b, :c] = np.arange(at[b], at[b] + c)
    order = torch.randperm(total + 8, generator=g, device="cuda").to(torch.int32)
    return order[torch.from_numpy(tables).cuda()].contiguous(), total + 8


def slots_of(tables, seq, pos):
    """The cache slots of positions `pos` of sequences `seq`."""
    return (tables[seq, pos // BLOCK] * BLOCK + pos % BLOCK).to(torch.int32)


def new_cache(case, blocks):
    """The 4-bit cache of one layer that a program keeps: the framework's, or plain tensors."""
    if own:
        import gollmgo_amd.verify as gv
        from gollmgo_amd._lib import DType
        return gv.KVCache(1, blocks, BLOCK, case["kv_heads"], case["dim"], DType.INT4)
    h, d, n = case["kv_heads"], case["dim"], blocks * BLOCK
    return {"k": torch.zeros(n, h, d // 2, dtype=torch.uint8, device="cuda"), "k_s": torch.zeros(n, h, device="cuda"),
            "k_z": torch.zeros(n, h, dtype=torch.uint8, device="cuda"),
            "v": torch.zeros(n, h, d // 2, dtype=torch.uint8, device="cuda"), "v_s": torch.zeros(n, h, device="cuda"),
            "v_z": torch.zeros(n, h, dtype=torch.uint8, device="cuda")}


def new_workspace(kv, out, tables):
    """The scratch memory a program keeps for the attention; the plain form needs none."""
    return kv.attention_workspace(out.shape[0], out.shape[1], out.shape[2], tables.shape[1]) if own else None


def write(kv, k, v, slots):
    if own:
        kv.append(0, k, v, slots)
    else:
        plain_write(kv, k, v, slots)


def prepare(case, seed):
    g = generator(seed)
    kind = case["kind"]
    if kind in ("rope", "rope_kv"):
        n = case["tokens"]
        s = projected(case, g, n)
        pos = torch.arange(n, device="cuda") + case["far"]
        axes = [pos if a == 0 else torch.randint(0, 64, (n,), generator=g, device="cuda") for a in range(case["axes"])]
        s["positions"] = torch.stack(axes).to(torch.int32).contiguous()
        if kind == "rope_kv":
            tables, blocks = blocks_for(g, [(n + BLOCK - 1) // BLOCK])
            at = torch.arange(n, device="cuda")
            s["slots"] = slots_of(tables, torch.zeros_like(at), at)
            s["kv"] = new_cache(case, blocks)
        s["case"] = case
        return s
    if kind == "cache":
        n, first = case["tokens"], case["first"]
        tables, blocks = blocks_for(g, [(first % BLOCK + n + BLOCK - 1) // BLOCK])
        at = torch.arange(n, device="cuda") + first % BLOCK
        k, v = cached_rows(case, g, n)
        return {"case": case, "k": k, "v": v, "slots": slots_of(tables, torch.zeros_like(at), at), "kv": new_cache(case, blocks)}
    ctx, rows = lengths(case)
    keys = ctx + rows
    tables, blocks = blocks_for(g, (keys + BLOCK - 1) // BLOCK)
    kv = new_cache(case, blocks)
    filled = keys if kind == "attention" else ctx  # a layer's own rows come with the call
    seq = torch.from_numpy(np.repeat(np.arange(case["seqs"]), filled)).cuda()
    first = torch.from_numpy(np.concatenate([[0], np.cumsum(filled)[:-1]])).cuda()
    pos = torch.arange(int(filled.sum()), device="cuda") - first[seq]
    k, v = cached_rows(case, g, int(filled.sum()))
    write(kv, k, v, slots_of(tables, seq, pos))
    s = {"case": case, "kv": kv, "tables": tables, "ctx_lens": torch.from_numpy(keys.astype(np.int32)).cuda(),
         "row_counts": torch.from_numpy(rows.astype(np.int32)).cuda(), "scale": 1.0 / math.sqrt(case["dim"])}
    B, R = case["seqs"], case["rows"]
    if kind == "layer":
        s.update(projected(case, g, B * R))
        j = torch.arange(R, device="cuda")
        at = torch.from_numpy(ctx).cuda()[:, None] + j[None, :]
        live = j[None, :] < s["row_counts"][:, None]
        s["positions"] = at.reshape(1, B * R).to(torch.int32).contiguous()
        grid = torch.arange(B, device="cuda")[:, None].expand(B, R)
        cols = torch.minimum(at, s["ctx_lens"][:, None] - 1)
        s["slots"] = torch.where(live, slots_of(tables, grid, cols), -1).reshape(-1).to(torch.int32).contiguous()
        s["k_in"] = torch.zeros(B * R, case["kv_heads"], case["dim"], dtype=TORCH[case["io"]], device="cuda")
        s["v_in"] = torch.zeros_like(s["k_in"])
    else:
        s["q"] = (2.0 * normal(g, B, R, case["q_heads"], case["dim"])).to(TORCH[case["io"]])
    s["out"] = torch.zeros(B, R, case["q_heads"], case["dim"], dtype=TORCH[case["io"]], device="cuda")
    s["ws"] = new_workspace(kv, s["out"], tables)
    return s


def cached_rows(case, g, n):
    """Keys and values as a model's layer leaves them: keys with a few large channels."""
    h, d, io = case["kv_heads"], case["dim"], TORCH[case["io"]]
    k = normal(g, n, h, d)
    k[:, :, :: max(1, d // 4)] *= 3.0
    return k.to(io), (normal(g, n, h, d) * (0.3 + torch.rand(n, h, 1, generator=g, device="cuda"))).to(io)


# ---- one pass ----

def run(s):
    case = s["case"]
    if own:
        return run_own(s, case)
    kind = case["kind"]
    if kind in ("rope", "rope_kv"):
        q, k, v = split(case, s["qkv"])
        q_out, k_out = plain_rope(case, s, q, k)
        if kind == "rope":
            return {"q": q_out.to(q.dtype), "k": k_out.to(k.dtype)}
        plain_write(s["kv"], k_out, v, s["slots"])
        k_in, v_in = plain_read(s["kv"], s["slots"].long())
        return {"q": q_out.to(q.dtype), "k": k_in.to(k.dtype), "v": v_in.to(k.dtype)}
    if kind == "cache":
        plain_write(s["kv"], s["k"], s["v"], s["slots"])
        k, v = plain_read(s["kv"], s["slots"].long())
        return {"k": k.to(s["k"].dtype), "v": v.to(s["k"].dtype)}
    if kind == "layer":
        q, k, v = split(case, s["qkv"])
        q, k = plain_rope(case, s, q, k)
        q, k = q.to(v.dtype), k.to(v.dtype)
        live = s["slots"] >= 0
        plain_write(s["kv"], k[live], v[live], s["slots"][live])
        s["k_in"][live], s["v_in"][live] = (x.to(q.dtype) for x in plain_read(s["kv"], s["slots"][live].long()))
        return {"out": plain_attention(s, q.reshape(s["out"].shape)), "k": s["k_in"], "v": s["v_in"]}
    return {"out": plain_attention(s, s["q"])}


def plain_rope(case, s, q, k):
    angle = s["positions"].double()[axis_of_pair(case)] * s["freq"].double()[:, None]  # [pairs, tokens]
    cos, sin = angle.cos().float().T[:, None, :], angle.sin().float().T[:, None, :]
    n, pairs = s["freq"].numel(), case.get("pairs", False)

    def turned(x, weight):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
        a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if pairs else (x[..., :n], x[..., n:2 * n])
        a, b = a * cos - b * sin, b * cos + a * sin
        both = torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1)
        return torch.cat([both, x[..., 2 * n:]], -1)

    return turned(q, s["q_weight"]), turned(k, s["k_weight"])


def plain_codes(x):
    x = torch.nan_to_num(x.float(), nan=0.0).clamp(-1e36, 1e36)
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0.0), x.amax(-1, keepdim=True).clamp(min=0.0)
    r = torch.true_divide(hi - lo, torch.full_like(lo, 15.0))
    s = ((r.view(torch.int32) + 0x7ffff) & -0x80000).view(torch.float32).clamp(min=2.0 ** -100)
    z = torch.round(-lo / s)
    return (torch.round(x / s) + z).clamp(0, 15).to(torch.uint8), s[..., 0], z[..., 0].to(torch.uint8)


def plain_write(kv, k, v, slots):
    at = slots.long()
    for name, x in (("k", k), ("v", v)):
        n, s, z = plain_codes(x)
        kv[name][at] = n[..., 0::2] | (n[..., 1::2] << 4)
        kv[name + "_s"][at], kv[name + "_z"][at] = s, z


def plain_read(kv, at):
    """The values of the slots `at` (any shape), keys and values [..., kv heads, dim]."""
    def values(name):
        p = kv[name][at]
        n = torch.stack([p & 15, p >> 4], -1).flatten(-2).float()
        return (n - kv[name + "_z"][at].float()[..., None]) * kv[name + "_s"][at][..., None]

    return values("k"), values("v")


def plain_attention(s, q):
    B, R, hq, d = q.shape
    tables, ctx, rows = s["tables"].long(), s["ctx_lens"].long(), s["row_counts"].long()
    t = torch.arange(tables.shape[1] * BLOCK, device="cuda")
    at = (tables[:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda")).flatten(1)  # [B, T]
    k, v = plain_read(s["kv"], at)  # [B, T, Hkv, D]
    h = k.shape[2]
    g = hq // h
    last = (ctx - rows)[:, None] + torch.arange(R, device="cuda")  # row j of a sequence sees keys up to here
    seen = t[None, None, :] <= last[:, :, None]  # [B, R, T]
    qh = q.float().view(B, R, h, g, d).permute(0, 2, 1, 3, 4).reshape(B, h, R * g, d)
    score = torch.matmul(qh, k.permute(0, 2, 3, 1).contiguous()) * s["scale"]
    score = score.masked_fill(~seen[:, None, :, None, :].expand(B, 1, R, g, t.numel()).reshape(B, 1, R * g, -1), -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous())
    o = o.view(B, h, R, g, d).permute(0, 2, 1, 3, 4).reshape(B, R, hq, d)
    live = torch.arange(R, device="cuda")[None, :] < rows[:, None]
    return torch.where(live[:, :, None, None], o, s["out"].float()).to(s["out"].dtype)


def run_own(s, case):
    import gollmgo_amd.verify as gv
    kind = case["kind"]
    if kind in ("rope", "rope_kv", "layer"):
        q, k, v = split(case, s["qkv"])
        turn = dict(positions=s["positions"], inv_freq=s["freq"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS,
                    pair_axis=axis_of_pair(case) if case.get("axes", 1) > 1 else None,
                    style="pairs" if case.get("pairs") else "halves")
        if kind == "rope_kv":
            q = s["kv"].norm_rope_append(0, q, k, v, slot_mapping=s["slots"], **turn)
            k, v = s["kv"].read(0, s["slots"], dtype=q.dtype)
            return {"q": q, "k": k, "v": v}
        q, k = gv.qk_norm_rope(q, k, **turn)
        if kind == "rope":
            return {"q": q, "k": k}
        s["kv"].attention_plan(s["ctx_lens"], case["rows"], case["q_heads"], s["tables"].shape[1], s["ws"], row_counts=s["row_counts"])
        out = s["kv"].append_attention(0, k, v.contiguous(), q.view(s["out"].shape), s["out"], s["ctx_lens"], s["tables"], s["scale"],
                                       s["ws"], row_counts=s["row_counts"])
        k, v = s["kv"].read(0, s["slots"], out=(s["k_in"], s["v_in"]))
        return {"out": out, "k": k, "v": v}
    if kind == "cache":
        s["kv"].append(0, s["k"], s["v"], s["slots"])
        k, v = s["kv"].read(0, s["slots"], dtype=s["k"].dtype)
        return {"k": k, "v": v}
    s["kv"].attention_plan(s["ctx_lens"], case["rows"], case["q_heads"], s["tables"].shape[1], s["ws"], row_counts=s["row_counts"])
    return {"out": s["kv"].attention(0, s["q"], s["out"], s["ctx_lens"], s["tables"], s["scale"], row_counts=s["row_counts"],
                                     workspace=s["ws"], planned=True)}


# ---- the definition in 64 bits ----

def exact_values(x):
    """What rows x [..., dim] stand for after 4-bit quantisation, with numbers of 64 bits: the
    scale's rounding up to five significant bits by its exponent."""
    x = x.double()
    top = torch.clamp(x.max(-1).values, min=0)
    low = torch.clamp(x.min(-1).values, max=0)
    step = (top - low) / 15
    mant, e = torch.frexp(step)
    step = torch.ldexp(torch.ceil(mant * 32) / 32, e).clamp(min=2.0 ** -100).unsqueeze(-1)
    zero = torch.round(-low.unsqueeze(-1) / step)
    return step * ((torch.round(x / step) + zero).clamp(0, 15) - zero)


def exact_turn(case, s, x, weight):
    """Normed and turned rows: each pair as a complex number times exp(i angle)."""
    x = x.double()
    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    n = s["freq"].numel()
    pos = torch.stack([s["positions"][a] for a in axis_of_pair(case)], -1).double()  # [tokens, pairs]
    turn = torch.polar(torch.ones_like(pos), pos * s["freq"].double())[:, None, :]
    if case.get("pairs"):
        y = torch.view_as_real(torch.view_as_complex(x[..., :2 * n].reshape(*x.shape[:-1], n, 2).contiguous()) * turn).flatten(-2)
    else:
        c = torch.complex(x[..., :n], x[..., n:2 * n]) * turn
        y = torch.cat([c.real, c.imag], -1)
    return torch.cat([y, x[..., 2 * n:]], -1)


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        kind = case["kind"]
        if kind in ("attention", "layer"):
            return exact_attention(case, seed)
        s = prepare(case, seed)
        if kind == "cache":
            return {"k": exact_values(s["k"]), "v": exact_values(s["v"])}
        q, k, v = split(case, s["qkv"])
        if kind == "rope":
            return {"q": exact_turn(case, s, q, s["q_weight"]), "k": exact_turn(case, s, k, s["k_weight"])}
        return {"q": exact_turn(case, s, q, s["q_weight"]), "k": exact_values(exact_turn(case, s, k, s["k_weight"])),
                "v": exact_values(v)}
    finally:
        own = kept


def exact_attention(case, seed):
    """Sequence by sequence and head by head over the rows as they were before quantisation."""
    s = prepare(case, seed)
    ctx, rows = lengths(case)
    keys = ctx + rows
    filled = keys if case["kind"] == "attention" else ctx
    g = generator(seed)
    blocks_for(g, (keys + BLOCK - 1) // BLOCK)  # the same draws, in the same order, as prepare
    k, v = cached_rows(case, g, int(filled.sum()))
    R, hq, h, d = case["rows"], case["q_heads"], case["kv_heads"], case["dim"]
    out = s["out"].double()
    at = np.concatenate([[0], np.cumsum(filled)])
    if case["kind"] == "layer":
        nq, nk, nv = split(case, s["qkv"])
        io = TORCH[case["io"]]
        nq, nk = exact_turn(case, s, nq, s["q_weight"]).to(io), exact_turn(case, s, nk, s["k_weight"]).to(io)
    for b in range(case["seqs"]):
        n = int(rows[b])
        kb, vb = k[at[b]:at[b + 1]], v[at[b]:at[b + 1]]
        if case["kind"] == "layer":
            kb, vb = torch.cat([kb, nk[b * R:b * R + n]]), torch.cat([vb, nv[b * R:b * R + n]])
            qb = nq[b * R:b * R + n].double()
        else:
            qb = s["q"][b, :n].double()
        kb, vb = exact_values(kb), exact_values(vb)
        hidden = torch.arange(keys[b], device="cuda")[None, :] > torch.arange(int(ctx[b]), int(keys[b]), device="cuda")[:, None]
        for i in range(hq):
            w = (qb[:, i] @ kb[:, i // (hq // h)].T.contiguous()) * s["scale"]
            w[hidden] = -math.inf
            out[b, :n, i] = torch.softmax(w, -1) @ vb[:, i // (hq // h)].contiguous()
    if case["kind"] == "attention":
        return {"out": out}
    live = (s["slots"] >= 0)[:, None, None]
    return {"out": out, "k": torch.where(live, exact_values(nk), 0.0), "v": torch.where(live, exact_values(nv), 0.0)}
