"""4-bit pools on the GPU: rows quantised on write bit for bit, read back, swapped, and attended
to, against the plain restatement (int4_ref)."""
import math

import numpy as np
import pytest
import torch

import int4_ref as ref
from gollmgo_amd._lib import DType, GGError
from helpers import say

pytestmark = pytest.mark.gpu
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def gv():
    import gollmgo_amd.verify as gv
    return gv


def rows_of(rng, n, h, d, kind="normal"):
    x = rng.normal(0, 1, (n, h, d)).astype(np.float32)
    if kind == "outliers":
        x[..., ::max(1, d // 3)] *= 9
    elif kind == "positive":
        x = np.abs(x) + 5
    elif kind == "constant":
        x[:] = -3.25
    elif kind == "zero":
        x[:] = 0
    elif kind == "wide":
        x *= np.exp2(rng.integers(-30, 31, (n, h, 1))).astype(np.float32)
    elif kind == "special":
        x[0, :, 0], x[min(1, n - 1), :, 1 % d], x[n // 2, :, 0], x[n // 2, :, d - 1] = np.nan, np.inf, -np.inf, np.inf
        x[n - 1] = np.nan
    return x


def to_dev(x, dt):
    t = torch.from_numpy(np.array(x, order="C")).to(TORCH[dt]).cuda()
    return t, t.float().cpu().numpy()


def check_pool(kv, layer, k, v, slots):
    """The written slots hold exactly the codes and scales of the rule."""
    nb, h, bs, d = kv.num_blocks, kv.num_kv_heads, kv.block_size, kv.head_dim
    kb = kv.k_pool(layer).cpu().numpy().reshape(nb, h, bs, d // 2)
    vb = kv.v_pool(layer).cpu().numpy().reshape(nb, h, d // 2, bs)
    (ks, kz), (vs, vz) = [[t.cpu().numpy() for t in p] for p in kv.scales(layer)]
    for x, s_dev, z_dev, got, pack in ((k, ks, kz, lambda b, o: kb[b, :, o], ref.pack_k),
                                       (v, vs, vz, lambda b, o: vb[b, :, :, o], ref.pack_v)):
        n, s, z = ref.quantise(x)
        want = pack(n)
        for r, slot in enumerate(slots):
            if 0 <= slot < nb * bs:
                b, o = divmod(int(slot), bs)
                np.testing.assert_array_equal(s_dev[b, :, o], s[r])
                np.testing.assert_array_equal(z_dev[b, :, o], z[r])
                np.testing.assert_array_equal(got(b, o), want[r])


@pytest.mark.parametrize("d,bs,h,n,src,kind", [
    (128, 16, 8, 5, "bf16", "normal"), (128, 16, 8, 200, "bf16", "outliers"), (128, 16, 2, 1, "f32", "normal"),
    (64, 16, 3, 77, "f16", "normal"), (64, 16, 8, 300, "f32", "wide"), (256, 16, 2, 40, "bf16", "positive"),
    (128, 16, 1, 64, "f16", "constant"), (128, 16, 4, 33, "bf16", "zero"), (128, 16, 2, 35, "f32", "special"),
    (64, 16, 2, 35, "bf16", "special"), (80, 16, 2, 50, "bf16", "normal"), (96, 8, 3, 61, "f16", "outliers"),
    (2, 16, 1, 9, "f32", "normal"), (34, 7, 5, 40, "bf16", "normal"), (512, 16, 1, 20, "bf16", "wide"), (130, 1, 2, 6, "f32", "normal"),
])
def test_append_is_the_rule(gv, d, bs, h, n, src, kind):
    say(f"int4 append d={d} bs={bs} h={h} n={n} {src} {kind}")
    rng = np.random.default_rng(d * 1000 + n)
    nb = (n + bs - 1) // bs + 3
    kv = gv.KVCache(2, nb, bs, h, d, DType.INT4)
    slots = rng.permutation(nb * bs)[:n].astype(np.int32)
    if n > 4:
        slots[1], slots[3] = -1, nb * bs  # skipped rows
    k, kf = to_dev(rows_of(rng, n, h, d, kind), src)
    v, vf = to_dev(rows_of(rng, n, h, d, kind)[::-1], src)
    kv.append(1, k, v, torch.from_numpy(slots).cuda())
    check_pool(kv, 1, kf, vf, slots)
    # A layer that was not written holds nothing; neither do slots that were not.
    (ks, _), (vs, _) = kv.scales(0)
    assert not ks.any() and not vs.any()
    free = np.setdiff1d(np.arange(nb * bs), slots)
    (ks, _), _ = kv.scales(1)
    assert not ks.cpu().numpy().swapaxes(1, 2).reshape(nb * bs, h)[free].any()
    kv.close()


@pytest.mark.parametrize("first,n,d", [(0, 64, 128), (0, 1000, 128), (5, 300, 128), (13, 19, 64), (0, 16, 128), (1, 15, 128), (0, 100, 256),
                                       (0, 100, 96), (5, 70, 80), (0, 40, 8), (3, 50, 200)])
def test_append_prompt_runs(gv, first, n, d):
    """Consecutive slots of whole and partial blocks of a shuffled table; neighbours in the first
    and last block keep their bytes."""
    say(f"int4 prompt first={first} n={n} d={d}")
    rng = np.random.default_rng(n + first)
    h, bs = 4, 16
    nblk = (first + n + bs - 1) // bs
    kv = gv.KVCache(1, nblk + 2, bs, h, d, DType.INT4)
    table = rng.permutation(nblk + 2)[:nblk]
    pos = np.arange(nblk * bs)
    all_slots = (table[pos // bs] * bs + pos % bs).astype(np.int32)
    k0, k0f = to_dev(rows_of(rng, nblk * bs, h, d), "bf16")
    kv.append(0, k0, k0, torch.from_numpy(all_slots).cuda())
    k, kf = to_dev(rows_of(rng, n, h, d, "outliers"), "bf16")
    v, vf = to_dev(rows_of(rng, n, h, d), "bf16")
    kv.append(0, k, v, torch.from_numpy(all_slots[first:first + n].copy()).cuda())
    wk, wv = k0f.copy(), k0f.copy()
    wk[first:first + n], wv[first:first + n] = kf, vf
    check_pool(kv, 0, wk, wv, all_slots)
    kv.close()


@pytest.mark.parametrize("src", ["bf16", "f16", "f32"])
def test_append_of_offset_views(gv, src):
    """Sources that are not 16-byte aligned."""
    rng = np.random.default_rng(9)
    n, h, d = 37, 2, 128
    kv = gv.KVCache(1, 4, 16, h, d, DType.INT4)
    base, bf = to_dev(rng.normal(0, 1, n * h * d + 1).astype(np.float32), src)
    k, kf = base[1:].view(n, h, d), bf[1:].reshape(n, h, d)
    slots = np.arange(n, dtype=np.int32) + 3
    kv.append(0, k, k, torch.from_numpy(slots).cuda())
    check_pool(kv, 0, kf, kf, slots)
    kv.close()


@pytest.mark.parametrize("pool,d,bs", [(DType.INT4, 128, 16), (DType.INT4, 64, 16), (DType.INT4, 34, 7), (DType.INT4, 256, 16),
                                       (DType.INT8, 128, 16), (DType.FP8_E4M3, 128, 16), (DType.BF16, 64, 16),
                                       (DType.F16, 80, 8), (DType.F32, 128, 16), (DType.INT4, 96, 16), (DType.INT4, 80, 16),
                                       (DType.INT4, 208, 16), (DType.INT4, 40, 16), (DType.INT4, 16, 8)])
@pytest.mark.parametrize("dst", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 50])
def test_read_gives_the_pool_back(gv, pool, d, bs, dst, n):
    say(f"read {pool.name} d={d} bs={bs} {dst} n={n}")
    rng = np.random.default_rng(n + d)
    h, nb = 3, 12
    kv = gv.KVCache(2, nb, bs, h, d, pool)
    if pool == DType.FP8_E4M3:
        kv.set_head_scales(1, [0.01, 0.02, 0.5], [0.02, 0.03, 0.125])
    slots = np.arange(n, dtype=np.int32) + 3
    k, kf = to_dev(rows_of(rng, n, h, d), "f32")
    v, vf = to_dev(rows_of(rng, n, h, d, "outliers"), "f32")
    kv.append(1, k, v, torch.from_numpy(slots).cuda())
    ask = np.concatenate([slots[::-1], [-1, nb * bs, slots[0]]]).astype(np.int32)
    ko = torch.full((len(ask), h, d), 7.0, dtype=TORCH[dst], device="cuda")
    vo = torch.full_like(ko, 7.0)
    kv.read(1, torch.from_numpy(ask).cuda(), out=(ko, vo))
    if pool == DType.INT4:
        K, V = ref.pool_values(kv, 1)
        wk, wv = [x.swapaxes(1, 2).reshape(nb * bs, h, d) for x in (K, V)]
    else:
        eb = {DType.INT8: 1, DType.FP8_E4M3: 1, DType.BF16: 2, DType.F16: 2, DType.F32: 4}[pool]
        view = {DType.INT8: torch.int8, DType.FP8_E4M3: torch.float8_e4m3fn, DType.BF16: torch.bfloat16,
                DType.F16: torch.float16, DType.F32: torch.float32}[pool]
        kp = kv.k_pool(1).view(view).view(nb, h, bs, d).float()
        vp = kv.v_pool(1).view(view).view(nb, h, d, bs).transpose(2, 3).float()
        if eb == 1:
            ks, vs = kv.scales(1)
            ks, vs = (ks[:h].view(1, h, 1, 1), vs[:h].view(1, h, 1, 1)) if pool == DType.FP8_E4M3 else (
                ks.float().view(nb, h, 1, 1), vs.float().view(nb, h, 1, 1))
            kp, vp = kp * ks, vp * vs
        wk, wv = [x.cpu().numpy().swapaxes(1, 2).reshape(nb * bs, h, d) for x in (kp, vp)]
    for got, want in ((ko, wk), (vo, wv)):
        got = got.cpu()
        ok = (ask >= 0) & (ask < nb * bs)
        want_t = torch.from_numpy(want[np.where(ok, ask, 0)]).float().to(TORCH[dst])  # (values are fp32 products)
        assert torch.equal(got[torch.from_numpy(ok)], want_t[torch.from_numpy(ok)])
        assert (got[torch.from_numpy(~ok)] == 7).all()
    only = torch.empty_like(ko)
    assert kv.read(1, torch.from_numpy(ask).cuda(), out=(None, only))[0] is None
    okc = torch.from_numpy(ok).cuda()
    assert torch.equal(only[okc], vo[okc])
    kv.close()


def test_read_refusals(gv):
    kv = gv.KVCache(1, 4, 16, 2, 64, DType.INT4)
    slots = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        kv.read(0, slots, out=(torch.empty(2, 2, 64, device="cuda"), None))
    with pytest.raises(ValueError):
        kv.read(0, slots, out=(None, None))
    with pytest.raises(TypeError):
        kv.read(0, slots, out=(torch.empty(3, 2, 64, device="cuda"), torch.empty(3, 2, 64, device="cuda").half()))
    with pytest.raises(TypeError):
        kv.read(0, slots, dtype=torch.int8)
    with pytest.raises(TypeError):
        kv.read(0, slots.long())
    with pytest.raises(GGError):
        kv.read(1, slots)
    k, v = kv.read(0, slots[:0])
    assert k.shape == (0, 2, 64)
    kv.close()


@pytest.mark.parametrize("d,bs,h", [(128, 16, 8), (34, 7, 3), (2, 1, 1)])
def test_snapshot_and_restore(gv, d, bs, h):
    say(f"int4 swap d={d} bs={bs}")
    rng = np.random.default_rng(3)
    nb = 9
    kv = gv.KVCache(2, nb, bs, h, d, DType.INT4)
    slots = torch.arange(nb * bs, dtype=torch.int32, device="cuda")
    for layer in range(2):
        k, _ = to_dev(rows_of(rng, nb * bs, h, d), "bf16")
        kv.append(layer, k, k.flip(0).contiguous(), slots)
    before = [ref.pool_values(kv, layer) for layer in range(2)]
    ids = torch.tensor([4, 1, 7], dtype=torch.int32, device="cuda")
    host = torch.empty(kv.snapshot_bytes(3), dtype=torch.uint8, pin_memory=True)
    staging, _ = kv.snapshot(ids, host=host)
    torch.cuda.synchronize()
    to = torch.tensor([0, 4, 2], dtype=torch.int32, device="cuda")
    kv.restore(to, staging, host=host)
    for layer in range(2):
        for got, want in zip(ref.pool_values(kv, layer), before[layer]):
            expect = want.copy()
            expect[[0, 4, 2]] = want[[4, 1, 7]]
            np.testing.assert_array_equal(got, expect)
    kv.close()


# ---- attention ----

def filled(gv, rng, ctx, h, d, bs, max_blocks=None, kind="normal", layers=1, spare=3):
    """A pool with `ctx` tokens of each sequence in shuffled blocks; tables padded with -1."""
    need = [(max(int(c), 0) + bs - 1) // bs for c in ctx]
    nb = sum(need) + spare
    order = rng.permutation(nb)
    mb = max_blocks or max(max(need), 1)
    tables = np.full((len(ctx), mb), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :min(n, mb)] = order[at:at + n][:mb]
        at += n
    kv = gv.KVCache(layers, nb, bs, h, d, DType.INT4)
    every = torch.arange(nb * bs, dtype=torch.int32, device="cuda")
    for layer in range(layers):  # (slots behind a sequence's end hold stale rows)
        k, _ = to_dev(rows_of(rng, nb * bs, h, d, kind), "bf16")
        v, _ = to_dev(rows_of(rng, nb * bs, h, d, kind), "bf16")
        kv.append(layer, k, v, every)
    return kv, tables


SHAPES = [
    # d, bs, Hq, H, R, contexts, row counts (None: all)
    (128, 16, 8, 2, 1, [1, 2, 17, 200], None),
    (128, 16, 32, 8, 5, [5, 64, 65, 300, 1000], [5, 1, 3, 5, 4]),
    (128, 16, 24, 8, 6, [1500, 40], None),
    (128, 16, 8, 1, 9, [777, 9, 64], None),
    (128, 16, 4, 4, 2, [2, 3, 130], [2, 0, 3]),
    (64, 16, 8, 2, 5, [5, 257, 1200], None),
    (64, 16, 32, 2, 6, [700, 31], [6, 2]),
    (64, 16, 16, 2, 8, [900, 8, 33], [8, 8, 5]),
    (128, 16, 12, 2, 8, [1100, 9, 31], [8, 7, 1]),
    (80, 16, 4, 2, 3, [3, 100, 700], None),
    (96, 16, 6, 3, 2, [2, 65, 500], [2, 1, 2]), (128, 32, 4, 2, 2, [2, 70, 300], None), (120, 64, 4, 1, 2, [130, 5], None),
    (128, 8, 4, 2, 2, [2, 70], None),
    (256, 16, 2, 1, 2, [90, 600], None),
    (34, 7, 3, 3, 2, [2, 20], None),
]


@pytest.mark.parametrize("shape", SHAPES, ids=[f"d{s[0]}b{s[1]}q{s[2]}h{s[3]}r{s[4]}" for s in SHAPES])
@pytest.mark.parametrize("io", ["bf16", "f16", "f32", "bf16-f32"])
def test_attention(gv, shape, io):
    d, bs, hq, h, R, ctx, rows = shape
    qdt, odt = io.split("-") if "-" in io else (io, io)
    say(f"int4 attention {shape} {io}")
    rng = np.random.default_rng(d + hq + R)
    kv, tables = filled(gv, rng, ctx, h, d, bs)
    check_attention(gv, kv, tables, rng, ctx, rows, R, hq, qdt, odt)
    kv.close()


def check_attention(gv, kv, tables, rng, ctx, rows, R, hq, qdt="bf16", odt="bf16", scale=None, partition=0, q=None, layer=0,
                    **kw):
    d = kv.head_dim
    B = len(ctx)
    q = rng.normal(0, 1.5, (B, R, hq, d)) if q is None else q
    qd, qf = to_dev(q.astype(np.float32), qdt)
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.full((B, R, hq, d), 11.0, dtype=TORCH[odt], device="cuda")
    cd = torch.from_numpy(np.asarray(ctx, np.int32)).cuda()
    rd = torch.from_numpy(np.asarray(rows, np.int32)).cuda() if rows is not None else None
    kv.attention(layer, qd, out, cd, torch.from_numpy(tables).cuda(), scale, row_counts=rd, partition_tokens=partition, **kw)
    K, V, k_span, v_span = ref.pool_values(kv, layer, spans=True)
    want, mag, reach, least = ref.attention(qf.astype(np.float64), K, V, ctx, rows if rows is not None else [R] * B, tables, scale,
                                            np.full(q.shape, 11.0), v_span)
    got = out.double().cpu().numpy()
    tol = ref.attention_tolerance(qf.astype(np.float64), K, k_span, scale, want, mag, reach, least, qdt, odt)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
    return got


@pytest.mark.parametrize("d,hq,h,R,ctx,wide", [
    (128, 9, 3, 8, [230, 238, 200, 31], None), (128, 3, 1, 4, [20] * 21, None), (128, 8, 2, 5, [1500, 700], 100),
    (128, 8, 1, 6, [1200, 90], 100), (64, 8, 2, 5, [300, 1700], 110), (64, 16, 2, 8, [900, 33], 80)])
@pytest.mark.parametrize("qdt", ["f32", "bf16"])
def test_attention_fp32_outputs_in_norm(gv, d, hq, h, R, ctx, wide, qdt):
    """The 2-norm of the error against 64 bits, which the largest deviations above do not bound closely.
    An exponent's argument lies below 2^5: half a step of 2^-20, evenly spread 2^-20 ln 2 / sqrt(3) =
    3.8e-7 of a probability; queries and probabilities to 22 bits and fp32 sums of products add less. Four
    times that."""
    say(f"int4 attention in norm d={d} q={hq}/{h} R={R} {ctx} {qdt}")
    rng = np.random.default_rng(d + sum(ctx))
    kv, tables = filled(gv, rng, ctx, h, d, 16, max_blocks=wide)
    q = rng.normal(0, 1.5, (len(ctx), R, hq, d)).astype(np.float32)
    qd, qf = to_dev(q, qdt)
    out = torch.zeros(q.shape, device="cuda")
    kv.attention(0, qd, out, torch.from_numpy(np.asarray(ctx, np.int32)).cuda(), torch.from_numpy(tables).cuda(), 1 / math.sqrt(d))
    K, V, _, v_span = ref.pool_values(kv, 0, spans=True)
    want = ref.attention(qf.astype(np.float64), K, V, ctx, [R] * len(ctx), tables, 1 / math.sqrt(d), np.zeros(q.shape), v_span)[0]
    assert np.linalg.norm(out.double().cpu().numpy() - want) <= 1.5e-6 * np.linalg.norm(want)
    kv.close()


@pytest.mark.parametrize("d,hq,h,R,ctx", [(128, 4, 1, 4, 60000), (64, 4, 2, 9, 24041), (128, 6, 1, 6, 30000), (128, 2, 2, 1, 40000)])
@pytest.mark.parametrize("io", ["f16", "bf16"])
def test_attention_long_contexts_in_norm(gv, d, hq, h, R, ctx, io):
    """Over many keys the sums of codes and of zero points grow and their difference averages out. The
    2-norm of the error against 64 bits: the output's rounding, and that of f16 probabilities, which for
    values of either sign weighs as much as rounding f16 outputs: sqrt(2) of the f16 output's, less of the
    bf16 one's. Half more than the output's own."""
    say(f"int4 attention long d={d} q={hq}/{h} R={R} {ctx} {io}")
    rng = np.random.default_rng(d + ctx)
    kv, tables = filled(gv, rng, [ctx], h, d, 16)
    qd, qf = to_dev(rng.normal(0, 1.5, (1, R, hq, d)).astype(np.float32), io)
    out = torch.zeros(qd.shape, dtype=TORCH[io], device="cuda")
    kv.attention(0, qd, out, torch.tensor([ctx], dtype=torch.int32, device="cuda"), torch.from_numpy(tables).cuda(), 1 / math.sqrt(d))
    K, V, _, v_span = ref.pool_values(kv, 0, spans=True)
    want = ref.attention(qf.astype(np.float64), K, V, [ctx], [R], tables, 1 / math.sqrt(d), np.zeros(qd.shape), v_span)[0]
    least = np.linalg.norm(torch.from_numpy(want).to(TORCH[io]).double().numpy() - want)
    assert np.linalg.norm(out.double().cpu().numpy() - want) <= 1.5 * least
    kv.close()


@pytest.mark.parametrize("partition", [64, 128, 1024])
def test_attention_partitions(gv, partition):
    rng = np.random.default_rng(1)
    ctx = [700, 65, 64, 3]
    kv, tables = filled(gv, rng, ctx, 2, 128, 16)
    check_attention(gv, kv, tables, rng, ctx, None, 3, 8, partition=partition)
    kv.close()


@pytest.mark.parametrize("wide", [None, 80])  # (a table past 512 keys: by pieces)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_holes_in_the_table(gv, d, wide):
    """Blocks missing from a table (negative ids, ids past the pool) hide their keys; a row that
    sees no key at all gives zeros."""
    rng = np.random.default_rng(2)
    ctx = [400, 100, 40, 17]
    kv, tables = filled(gv, rng, ctx, 2, d, 16, wide)
    tables[0, 3], tables[0, 10], tables[0, 24] = -1, kv.num_blocks, -7
    tables[1, :] = -1
    tables[2, 0] = 1 << 20
    tables[3, 0] = -1  # (rows 0.. see only the second block's one key, or none)
    got = check_attention(gv, kv, tables, rng, ctx, None, 3, 4)
    assert (got[1] == 0).all()
    kv.close()


@pytest.mark.parametrize("wide", [None, 80])
def test_attention_no_rows_and_no_keys(gv, wide):
    rng = np.random.default_rng(4)
    ctx = [0, -5, 2, 50]
    kv, tables = filled(gv, rng, [16, 16, 16, 50], 2, 128, 16, wide)
    check_attention(gv, kv, tables, rng, ctx, [2, 2, 3, 0], 3, 4)  # all: nothing to write
    kv.close()


@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-35])
def test_attention_scales(gv, scale):
    rng = np.random.default_rng(5)
    ctx = [300, 9]
    kv, tables = filled(gv, rng, ctx, 2, 128, 16)
    check_attention(gv, kv, tables, rng, ctx, None, 2, 4, scale=scale)
    kv.close()


@pytest.mark.parametrize("kind", ["outliers", "positive", "zero", "constant"])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_over_other_rows(gv, kind, d):
    rng = np.random.default_rng(6)
    ctx = [333, 1200]
    kv, tables = filled(gv, rng, ctx, 2, d, 16, kind=kind)
    check_attention(gv, kv, tables, rng, ctx, None, 2, 8, "f32", "f32", scale=0.02)
    kv.close()


@pytest.mark.parametrize("wide", [None, 80])
@pytest.mark.parametrize("odt", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_value_scales_far_apart(gv, d, odt, wide):
    """Tokens whose values differ by 2^60: a token hidden from a row, or nearly unweighted, must
    not cost the others their digits."""
    rng = np.random.default_rng(7)
    ctx, h, R = [200, 70], 2, 4
    kv, tables = filled(gv, rng, ctx, h, d, 16, wide)
    slots = np.concatenate([tables[b, np.arange(c) // 16] * 16 + np.arange(c) % 16 for b, c in enumerate(ctx)]).astype(np.int32)
    k, _ = to_dev(rows_of(rng, sum(ctx), h, d), "bf16")
    v = rows_of(rng, sum(ctx), h, d)
    v[199] *= 2.0 ** 40   # sequence 0's last row: hidden from rows 0..2
    v[200:220] *= 2.0 ** -20
    vd, _ = to_dev(v, "bf16")
    kv.append(0, k, vd, torch.from_numpy(slots).cuda())
    check_attention(gv, kv, tables, rng, ctx, None, R, 8, "bf16", odt)
    kv.close()


@pytest.mark.parametrize("wide", [None, 80])
@pytest.mark.parametrize("qdt", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_queries_of_any_size(gv, d, qdt, wide):
    """Rows of one item whose sizes lie far apart, a row of zeros, and one with a NaN or an
    infinity: each row as if it were alone."""
    rng = np.random.default_rng(8)
    ctx, R, hq = [150], 4, 4
    kv, tables = filled(gv, rng, ctx, 1, d, 16, wide)
    q = rng.normal(0, 1, (1, R, hq, d))
    q[0, 0] *= 2.0 ** -60
    q[0, 1] *= 2.0 ** 6
    q[0, 2, 1] = 0
    check_attention(gv, kv, tables, rng, ctx, None, R, hq, qdt, "f32", q=q)
    alone = check_attention(gv, kv, tables, rng, ctx, None, R, hq, qdt, "f32", q=q)
    bad = q.copy()
    bad[0, 3, 0, 5], bad[0, 3, 2, 7] = np.nan, np.inf
    qd, _ = to_dev(bad.astype(np.float32), qdt)
    out = torch.zeros(1, R, hq, d, device="cuda")
    kv.attention(0, qd, out, torch.tensor(ctx, dtype=torch.int32).cuda(), torch.from_numpy(tables).cuda(), 1 / math.sqrt(d))
    got = out.cpu().numpy()
    assert np.isnan(got[0, 3, 0]).all() and np.isnan(got[0, 3, 2]).all()
    keep = np.ones((R, hq), bool)
    keep[3, 0] = keep[3, 2] = False
    np.testing.assert_array_equal(got[0][keep], alone[0][keep].astype(np.float32))
    kv.close()


@pytest.mark.parametrize("d,hq,h,R,ctx,rows", [
    (128, 32, 8, 5, [5, 20, 300, 1000, 64], [5, 1, 3, 5, 4]), (128, 8, 1, 9, [9, 900], None), (64, 8, 2, 4, [4, 33, 500], None),
    (128, 16, 2, 12, [700, 12], None), (80, 4, 2, 3, [3, 90], None), (128, 8, 2, 20, [500, 20], None)])
@pytest.mark.parametrize("wide", [None, 80])
@pytest.mark.parametrize("src", ["bf16", "f32"])
def test_append_attention_equals_the_two_calls(gv, d, hq, h, R, ctx, rows, src, wide):
    say(f"int4 append+attention d={d} hq={hq} h={h} R={R} {ctx} {src}")
    rng = np.random.default_rng(R)
    B = len(ctx)
    pools = []
    for _ in range(2):
        pools.append(filled(gv, np.random.default_rng(11), ctx, h, d, 16, wide))
    (kv1, tables), (kv2, _) = pools
    counts = np.asarray(rows if rows is not None else [R] * B, np.int32)
    k, kf = to_dev(rows_of(rng, B * R, h, d, "outliers"), src)
    v, vf = to_dev(rows_of(rng, B * R, h, d), src)
    q, _ = to_dev(rng.normal(0, 1, (B, R, hq, d)).astype(np.float32), "bf16")
    cd, rd, td = torch.tensor(ctx, dtype=torch.int32).cuda(), torch.from_numpy(counts).cuda(), torch.from_numpy(tables).cuda()
    slots = np.full((B, R), -1, np.int32)
    for b in range(B):
        p = ctx[b] - counts[b] + np.arange(counts[b])
        slots[b, :counts[b]] = tables[b, p // 16] * 16 + p % 16
    o1, o2 = (torch.full((B, R, hq, d), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ws1, ws2 = (kv.attention_workspace(B, R, hq, tables.shape[1]) for kv in (kv1, kv2))
    kv1.attention_plan(cd, R, hq, tables.shape[1], ws1, row_counts=rd)
    kv2.attention_plan(cd, R, hq, tables.shape[1], ws2, row_counts=rd)
    kv1.append_attention(0, k, v, q, o1, cd, td, 0.1, ws1, row_counts=rd)
    kv2.append(0, k, v, torch.from_numpy(slots.reshape(-1)).cuda())
    kv2.attention(0, q, o2, cd, td, 0.1, row_counts=rd, workspace=ws2, planned=True)
    for a, b in zip(ref.pool_values(kv1), ref.pool_values(kv2)):
        np.testing.assert_array_equal(a, b)
    assert torch.equal(o1, o2)
    check_pool(kv1, 0, kf, vf, slots.reshape(-1))
    kv1.close(), kv2.close()


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d,R,hq,h", [(64, 5, 16, 4), (128, 5, 16, 4), (128, 1, 16, 2), (128, 9, 10, 2), (64, 8, 8, 1)])
def test_attention_whole_items(gv, d, R, hq, h, io):
    """Tables too narrow to cut and batches too large for the per-row kernel."""
    rng = np.random.default_rng(R)
    ctx = rng.integers(R, 350, 70)
    kv, tables = filled(gv, rng, ctx, h, d, 16)
    rows = rng.integers(1, R + 1, 70)
    check_attention(gv, kv, tables, rng, ctx, rows, R, hq, io, io)
    kv.close()


def test_attention_stale_slots(gv):
    """Rows behind a sequence's end, and in no block of its table, hold values 2^90 times larger: they
    change nothing."""
    rng = np.random.default_rng(21)
    ctx, h, d = [75, 130, 700], 2, 128
    kv, tables = filled(gv, rng, ctx, h, d, 16)
    every = np.arange(kv.num_blocks * 16)
    live = np.concatenate([tables[b, np.arange(c) // 16] * 16 + np.arange(c) % 16 for b, c in enumerate(ctx)])
    stale = np.setdiff1d(every, live).astype(np.int32)
    big, _ = to_dev(rows_of(rng, len(stale), h, d) * 2.0 ** 90, "bf16")
    kv.append(0, big, big, torch.from_numpy(stale).cuda())
    tables[1, 2] = -1
    for odt in ("bf16", "f32"):
        check_attention(gv, kv, tables, rng, ctx, None, 3, 8, "bf16", odt)
    kv.close()


def test_attention_many_sequences(gv):
    """More sequences than the plan ranks."""
    rng = np.random.default_rng(12)
    B = 1100
    ctx = rng.integers(1, 60, B)
    ctx[3] = 900
    kv, tables = filled(gv, rng, ctx, 1, 64, 16)
    check_attention(gv, kv, tables, rng, ctx, None, 1, 2)
    kv.close()


def test_graph_replays_a_layer(gv):
    """Plan, append and attention, read back: captured once, replayed with eager work between."""
    rng = np.random.default_rng(13)
    B, R, hq, h, d = 3, 4, 8, 2, 128
    ctx = [900, 70, 1500]
    kv, tables = filled(gv, rng, ctx, h, d, 16)
    cd, td = torch.tensor(ctx, dtype=torch.int32).cuda(), torch.from_numpy(tables).cuda()
    ws = kv.attention_workspace(B, R, hq, tables.shape[1])
    q = torch.zeros(B, R, hq, d, dtype=torch.bfloat16, device="cuda")
    k, v = (torch.zeros(B * R, h, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    out = torch.zeros_like(q)
    slots = torch.arange(5, dtype=torch.int32, device="cuda")
    back = tuple(torch.zeros(5, h, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def layer(ws, out, back):
        kv.attention_plan(cd, R, hq, tables.shape[1], ws)
        kv.append_attention(0, k, v, q, out, cd, td, 0.1, ws)
        kv.read(0, slots, out=back)

    layer(ws, out, back)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        layer(ws, out, back)
    for i in range(4):
        x = torch.from_numpy(rng.normal(0, 1, q.shape).astype(np.float32)).cuda()
        q.copy_(x)
        k.copy_(torch.from_numpy(rng.normal(0, 1, k.shape).astype(np.float32)))
        v.copy_(torch.from_numpy(rng.normal(0, 1, k.shape).astype(np.float32)))
        g.replay()
        got, gb = out.clone(), [t.clone() for t in back]
        eo, eb = torch.zeros_like(out), tuple(torch.zeros_like(t) for t in back)
        layer(torch.empty_like(ws), eo, eb)
        torch.cuda.synchronize()
        assert torch.equal(got, eo) and torch.equal(gb[0], eb[0]) and torch.equal(gb[1], eb[1])
    kv.close()


def test_streams_and_noalloc(gv):
    from gollmgo_amd._lib import check, lib
    rng = np.random.default_rng(14)
    ctx = [500, 40]
    kv, tables = filled(gv, rng, ctx, 2, 128, 16)
    q, _ = to_dev(rng.normal(0, 1, (2, 3, 4, 128)).astype(np.float32), "bf16")
    cd, td = torch.tensor(ctx, dtype=torch.int32).cuda(), torch.from_numpy(tables).cuda()
    a, b, c = (torch.zeros_like(q) for _ in range(3))
    kv.attention(0, q, a, cd, td, 0.1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    kv.attention(0, q, b, cd, td, 0.1, stream=s)
    s.synchronize()
    check(lib().gg_verify_attention_noalloc(kv.handle, 0, q.data_ptr(), int(DType.BF16), c.data_ptr(), int(DType.BF16),
                                            cd.data_ptr(), None, td.data_ptr(), tables.shape[1], 2, 3, 4, 0.1, None), "noalloc")
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(a, c)
    kv.close()


def test_offsets_past_32_bits(gv):
    """Blocks past 4 GiB of a pool: written, read and attended to as the same rows in a small pool."""
    say("int4 pool past 4 GiB")
    rng = np.random.default_rng(31)
    h, d, nb = 8, 128, 300_000
    ctx, R, hq = [700, 40, 1300], 3, 16
    small, tables = filled(gv, rng, ctx, h, d, 16)
    far = np.where(tables >= 0, nb - 1 - tables, -1).astype(np.int32)
    big = gv.KVCache(1, nb, 16, h, d, DType.INT4)
    n = small.num_blocks * 16
    k, _ = to_dev(rows_of(rng, n, h, d), "bf16")
    v, _ = to_dev(rows_of(rng, n, h, d), "bf16")
    slots = np.arange(n, dtype=np.int32)
    far_slots = ((nb - 1 - slots // 16) * 16 + slots % 16).astype(np.int32)
    sd, fd = torch.from_numpy(slots).cuda(), torch.from_numpy(far_slots).cuda()
    for kv, s in ((small, sd), (big, fd)):
        kv.append(0, k, v, s)
    for a, b in zip(small.read(0, sd), big.read(0, fd)):
        assert torch.equal(a, b)
    q, _ = to_dev(rng.normal(0, 1, (3, R, hq, d)).astype(np.float32), "bf16")
    cd = torch.tensor(ctx, dtype=torch.int32).cuda()
    o1, o2 = torch.zeros_like(q), torch.zeros_like(q)
    small.attention(0, q, o1, cd, torch.from_numpy(tables).cuda(), 0.1)
    big.attention(0, q, o2, cd, torch.from_numpy(far).cuda(), 0.1)
    assert torch.equal(o1, o2) and o1.abs().sum() > 0
    o3, o4 = torch.zeros_like(q), torch.zeros_like(q)  # the per-row kernel
    small.attention(0, q, o3, cd, torch.from_numpy(tables).cuda(), 0.1, partition_tokens=512)
    big.attention(0, q, o4, cd, torch.from_numpy(far).cuda(), 0.1, partition_tokens=512)
    assert torch.equal(o3, o4)
    small.close(), big.close()
