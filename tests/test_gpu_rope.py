"""Norm and rotation of query and key heads on the GPU, to dense rows and into pools of every type,
against float64."""
import numpy as np
import pytest
import torch

import int4_ref
from gollmgo_amd._lib import DType, GGError
from helpers import say

pytestmark = pytest.mark.gpu
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


@pytest.fixture(scope="module")
def gv():
    import gollmgo_amd.verify as gv
    return gv


def want(x, w, eps, pos, axis, freq, style):
    """The rows in float64 (angles in long double), and what an element's error is relative to."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    P = len(freq)
    mag = np.abs(x)
    if P:
        th = pos[axis].T.astype(np.longdouble) * freq.astype(np.longdouble)  # [n, P]
        c, s = np.cos(th).astype(np.float64)[:, None], np.sin(th).astype(np.float64)[:, None]
        ia, ib = (np.arange(0, 2 * P, 2), np.arange(1, 2 * P, 2)) if style == "pairs" else (np.arange(P), np.arange(P, 2 * P))
        a, b = x[..., ia], x[..., ib]
        x, mag = x.copy(), mag.copy()
        x[..., ia], x[..., ib] = a * c - b * s, b * c + a * s
        mag[..., ia] = mag[..., ib] = np.abs(a) + np.abs(b)
    return x, mag


def tolerance(ref, mag, d, far, dt):
    """fp32 sums of d squares (d 2^-24 relative, half of it in the root), six fp32 products and sums,
    cosines to 2^-22; angles in 64 bits: far * 2^-50; the output's half step."""
    return mag * (d * 2.0 ** -25 + 2.0 ** -20 + far * 2.0 ** -50) + HALF[dt] * np.abs(ref) + (2.0 ** -25 if dt == "f16" else 1e-37)


def inputs(rng, n, hq, hk, d, dt, P, axes, far):
    """Rows as slices of one projection of q, k and v heads."""
    x = rng.normal(0, 1, (n, hq + 2 * hk, d)) * np.exp2(rng.integers(-6, 7, (n, hq + 2 * hk, 1)))
    fused = torch.from_numpy(x.astype(np.float32)).to(TORCH[dt]).cuda()
    w = [torch.from_numpy((1 + 0.3 * rng.normal(0, 1, d)).astype(np.float32)).to(TORCH[dt]).cuda() for _ in range(2)]
    pos = rng.integers(0, 100, (axes, n)).astype(np.int32)
    pos[0] = far + np.arange(n)
    freq = (10000.0 ** (-np.arange(P) / max(P, 1))).astype(np.float32)
    axis = np.sort(rng.integers(0, axes, P))
    return fused, w, pos, freq, axis


def as_np(t):
    return t.float().cpu().numpy()


CASES = [
    # n, Hq, Hkv, D, pairs, axes, far, style
    (1, 32, 8, 128, 64, 1, 3001, "halves"), (5, 32, 8, 128, 64, 1, 0, "halves"), (300, 24, 8, 128, 64, 3, 5000, "halves"),
    (70, 8, 2, 64, 32, 1, 1000000, "halves"), (33, 4, 4, 128, 64, 2, 0, "pairs"), (9, 5, 1, 256, 128, 1, 77, "halves"),
    (17, 3, 3, 128, 32, 1, 9, "halves"), (17, 3, 1, 128, 16, 4, 9, "pairs"), (40, 7, 1, 80, 40, 1, 2, "halves"),
    (12, 2, 2, 34, 17, 1, 5, "halves"), (12, 2, 1, 34, 5, 2, 5, "pairs"), (8, 2, 1, 33, 0, 1, 0, "halves"), (3, 1, 1, 2, 1, 1, 4, "pairs"),
    (4, 2, 1, 1024, 512, 8, 2 ** 31 - 9, "halves"), (50, 16, 0, 128, 64, 1, 0, "halves"), (50, 0, 8, 64, 32, 1, 12, "halves"),
    (2000, 8, 2, 128, 64, 1, 0, "halves"), (19, 6, 2, 96, 24, 3, 1, "halves"), (4, 9, 3, 192, 96, 2, 30, "halves"),
]


@pytest.mark.parametrize("case", CASES, ids=["-".join(map(str, c)) for c in CASES])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_norm_rope(gv, case, dt):
    n, hq, hk, d, P, axes, far, style = case
    say(f"norm_rope {case} {dt}")
    rng = np.random.default_rng(n * 7 + d)
    fused, w, pos, freq, axis = inputs(rng, n, hq, hk, d, dt, P, axes, far)
    q, k = fused[:, :hq], fused[:, hq:hq + hk]
    kw = dict(positions=torch.from_numpy(pos).cuda(), inv_freq=torch.from_numpy(freq).cuda(), eps=1e-5,
              pair_axis=axis.tolist() if axes > 1 else None, style=style)
    for wq, wk in ((w[0], w[1]), (w[0], None), (None, None)):
        qo, ko = gv.qk_norm_rope(q if hq else None, k if hk else None, q_weight=wq, k_weight=wk, **kw)
        for x, o, weight in ((q, qo, wq), (k, ko, wk)):
            if not x.shape[1]:
                assert o is None
                continue
            ref, mag = want(as_np(x), None if weight is None else as_np(weight), 1e-5, pos, axis, freq, style)
            err = np.abs(as_np(o).astype(np.float64) - ref)
            tol = tolerance(ref, mag, d, abs(far) + n, dt)
            assert o.dtype == x.dtype and (err <= tol).all(), (np.argwhere(err > tol)[:4], err.max())


@pytest.mark.parametrize("d,P", [(128, 64), (64, 16), (80, 40)])
def test_norm_rope_in_place_and_unaligned(gv, d, P):
    """Outputs over the inputs; rows whose stride or base is not a multiple of a vector load."""
    rng = np.random.default_rng(3)
    n, hq, hk = 21, 4, 2
    fused, w, pos, freq, axis = inputs(rng, n, hq, hk, d, "bf16", P, 1, 40)
    kw = dict(positions=torch.from_numpy(pos).cuda(), inv_freq=torch.from_numpy(freq).cuda(), q_weight=w[0], k_weight=w[1])
    q, k = fused[:, :hq].contiguous(), fused[:, hq:hq + hk].contiguous()
    qo, ko = gv.qk_norm_rope(q, k, **kw)
    qi, ki = q.clone(), k.clone()
    a, b = gv.qk_norm_rope(qi, ki, q_out=qi, k_out=ki, **kw)
    assert a is qi and b is ki and torch.equal(qi, qo) and torch.equal(ki, ko)
    wide = torch.zeros(n, hq * d + 3, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:hq * d + 1] = q.view(n, -1)
    odd = torch.as_strided(wide, (n, hq, d), (hq * d + 3, d, 1), 1)
    qu, _ = gv.qk_norm_rope(odd, k, **kw)
    # (Another kernel: its sums run in another order.)
    ref, mag = want(as_np(q), as_np(w[0]), 1e-6, pos, axis, freq, "halves")
    assert (np.abs(as_np(qu) - ref) <= tolerance(ref, mag, d, 40 + n, "bf16")).all()


def test_norm_rope_special_rows(gv):
    """Zeros stay zero; a NaN or infinity keeps to its own head."""
    rng = np.random.default_rng(4)
    n, hq, hk, d, P = 6, 4, 2, 128, 64
    fused, w, pos, freq, axis = inputs(rng, n, hq, hk, d, "bf16", P, 1, 40)
    kw = dict(positions=torch.from_numpy(pos).cuda(), inv_freq=torch.from_numpy(freq).cuda(), q_weight=w[0], k_weight=w[1])
    clean, _ = gv.qk_norm_rope(fused[:, :hq], fused[:, hq:hq + hk], **kw)
    fused[1, 2] = 0
    fused[2, 1, 5], fused[3, 0, 7] = float("nan"), float("inf")
    got, _ = gv.qk_norm_rope(fused[:, :hq], fused[:, hq:hq + hk], **kw)
    assert (got[1, 2] == 0).all() and got[2, 1].isnan().all() and got[3, 0].isnan().any()
    same = torch.ones(n, hq, dtype=torch.bool, device="cuda")
    same[1, 2] = same[2, 1] = same[3, 0] = False
    assert torch.equal(got[same], clean[same])


POOLS = [DType.INT4, DType.FP8_E4M3, DType.BF16, DType.F16, DType.F32]
APPEND = [
    # n, Hq, Hkv, D, bs, pairs, axes, style, slots
    (1, 32, 8, 128, 16, 64, 1, "halves", "any"), (5, 32, 8, 128, 16, 64, 1, "halves", "run"), (90, 24, 8, 128, 16, 64, 3, "halves", "run"),
    (384, 8, 2, 128, 16, 64, 1, "halves", "any"), (64, 4, 2, 64, 16, 32, 1, "halves", "run"), (37, 4, 2, 64, 16, 32, 2, "pairs", "any"),
    (20, 2, 1, 256, 16, 128, 1, "halves", "run"), (33, 3, 3, 128, 16, 32, 1, "halves", "run"), (33, 0, 2, 128, 16, 64, 1, "pairs", "run"),
    (18, 4, 2, 80, 8, 40, 1, "halves", "any"), (9, 2, 1, 34, 7, 10, 1, "pairs", "any"), (50, 8, 4, 128, 16, 0, 1, "halves", "run5"),
    (70, 2, 3, 64, 16, 32, 1, "halves", "run"), (50, 2, 2, 256, 16, 128, 1, "halves", "run"), (50, 2, 1, 80, 16, 40, 1, "halves", "run"),
    (40, 1, 2, 24, 16, 8, 1, "pairs", "run"), (40, 1, 1, 160, 16, 64, 1, "halves", "run5"), (40, 2, 1, 8, 16, 4, 1, "halves", "run"),
]


@pytest.mark.parametrize("case", APPEND, ids=["-".join(map(str, c)) for c in APPEND])
@pytest.mark.parametrize("pool", POOLS, ids=[p.name for p in POOLS])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_norm_rope_append(gv, case, pool, dt):
    """q as qk_norm_rope gives it, bit for bit; the pool within its own half step of the rows in
    float64, and the values exactly as gg_kv_append writes them."""
    n, hq, h, d, bs, P, axes, style, how = case
    say(f"norm_rope_append {case} {pool.name} {dt}")
    rng = np.random.default_rng(n + d)
    fused, w, pos, freq, axis = inputs(rng, n, hq, h, d, dt, P, axes, 17)
    nb = (n + 5 + bs - 1) // bs + 2
    first = 5 if how == "run5" else 0
    slots = (rng.permutation(nb * bs)[:n] if how == "any" else
             (rng.permutation(nb)[(first + np.arange(n)) // bs] * bs + (first + np.arange(n)) % bs)).astype(np.int32)
    if n > 6:
        slots[2], slots[5] = -3, nb * bs
    q, k, v = fused[:, :hq], fused[:, hq:hq + h], fused[:, hq + h:]
    kw = dict(positions=torch.from_numpy(pos).cuda(), inv_freq=torch.from_numpy(freq).cuda(), q_weight=w[0], k_weight=w[1],
              pair_axis=axis.tolist() if axes > 1 else None, style=style)
    sd = torch.from_numpy(slots).cuda()
    kv, plain = (gv.KVCache(2, nb, bs, h, d, pool) for _ in range(2))
    if pool == DType.FP8_E4M3:
        for c in (kv, plain):
            c.set_head_scales(1, [0.02] * h, [0.2] * h)
    qo = kv.norm_rope_append(1, q if hq else None, k, v, slot_mapping=sd, **kw)
    if hq:
        assert torch.equal(qo, gv.qk_norm_rope(q, k, **kw)[0])
    else:
        assert qo is None
    ok = (slots >= 0) & (slots < nb * bs)
    live = torch.from_numpy(np.where(ok, slots, -1)).cuda()
    zero = lambda: torch.zeros(n, h, d, device="cuda")  # noqa: E731
    got_k, got_v = kv.read(1, live, out=(zero(), zero()))
    plain.append(1, k.contiguous(), v.contiguous(), sd)
    _, want_v = plain.read(1, live, out=(zero(), zero()))
    assert torch.equal(got_v, want_v)
    ref, mag = want(as_np(k), as_np(w[1]), 1e-6, pos, axis, freq, style)
    near = tolerance(ref, mag, d, 17 + n, "f32")
    if pool == DType.INT4:
        # Half a step: s = the row's range / 15, up to 1/16 longer, from rows that are off by `near`.
        rng_ = np.maximum(ref.max(-1), 0) - np.minimum(ref.min(-1), 0) + 2 * near.max(-1)
        tol = near + (rng_ / 15 * (1 + 1 / 16) / 2 * (1 + 2.0 ** -20))[..., None]
    elif pool == DType.FP8_E4M3:  # relative half step 2^-4, smallest 2^-10 of the scale, past 448 the end
        ref = np.clip(ref, -448 * 0.02, 448 * 0.02)
        tol = near * (1 + 2.0 ** -4) + 2.0 ** -4 * np.abs(ref) + 0.02 * 2.0 ** -10
    else:
        tol = near + {DType.BF16: HALF["bf16"], DType.F16: HALF["f16"], DType.F32: 0}[pool] * (np.abs(ref) + near) + (
            2.0 ** -25 if pool == DType.F16 else 0)
    err = np.abs(got_k.double().cpu().numpy() - ref)
    assert (err[ok] <= tol[ok]).all(), (np.argwhere(err > tol)[:4], err[ok].max())
    # Nothing else was written.
    assert (got_k[torch.from_numpy(~ok)] == 0).all()
    kv.close(), plain.close()


def test_norm_rope_append_int4_is_the_rule(gv):
    """Keys with no norm and no rotation go into a 4-bit pool as gg_kv_append writes them."""
    rng = np.random.default_rng(5)
    n, h, d = 70, 4, 128
    fused, w, pos, freq, axis = inputs(rng, n, 2, h, d, "bf16", 0, 1, 0)
    slots = torch.from_numpy(rng.permutation(96)[:n].astype(np.int32)).cuda()
    a, b = (gv.KVCache(1, 6, 16, h, d, DType.INT4) for _ in range(2))
    a.norm_rope_append(0, fused[:, :2], fused[:, 2:2 + h], fused[:, 2 + h:], torch.from_numpy(pos).cuda(),
                       torch.from_numpy(freq).cuda(), slots)
    b.append(0, fused[:, 2:2 + h].contiguous(), fused[:, 2 + h:].contiguous(), slots)
    for x, y in zip(int4_ref.pool_values(a), int4_ref.pool_values(b)):
        np.testing.assert_array_equal(x, y)
    a.close(), b.close()


def test_refusals(gv):
    n, hq, h, d = 4, 4, 2, 64
    q, k = torch.zeros(n, hq, d, device="cuda"), torch.zeros(n, h, d, device="cuda")
    pos, freq = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda")
    call = lambda **kw: gv.qk_norm_rope(**{**dict(q=q, k=k, positions=pos, inv_freq=freq), **kw})  # noqa: E731
    call()
    for bad in (dict(q=None, k=None), dict(k=k.half()), dict(k=k[:2]), dict(positions=pos[:2]), dict(style="spiral"),
                dict(positions=torch.stack([pos, pos])), dict(positions=torch.stack([pos, pos]), pair_axis=[0] * 31),
                dict(pair_axis=[1] * 32), dict(pair_axis=[-1] * 32), dict(q_weight=torch.ones(d, device="cuda").half()),
                dict(k_weight=torch.ones(d - 1, device="cuda")), dict(q=q.cpu(), k=k.cpu()), dict(q=q.transpose(1, 2)),
                dict(q_out=torch.zeros(1, device="cuda"))):
        with pytest.raises((ValueError, TypeError)):
            call(**bad)
    with pytest.raises(TypeError):
        call(positions=pos.long())
    with pytest.raises(GGError):
        call(inv_freq=torch.ones(33, device="cuda"))
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(GGError):
            call(eps=eps)
    with pytest.raises(GGError):
        call(q=q[:1].expand(n, hq, d))  # rows that overlap
    with pytest.raises(GGError):
        call(positions=torch.zeros(9, n, dtype=torch.int32, device="cuda"), pair_axis=[8] * 32)
    slots = torch.zeros(n, dtype=torch.int32, device="cuda")
    kv = gv.KVCache(1, 2, 16, h, d, DType.INT8)
    with pytest.raises(GGError, match="PER_BLOCK"):
        kv.norm_rope_append(0, q, k, k, pos, freq, slots)
    kv.close()
    kv = gv.KVCache(1, 2, 16, h, d, DType.INT4)
    for args in ((q, k, k[:, :1], pos, freq, slots), (q, k, k.half(), pos, freq, slots), (q, k, k, pos, freq, slots[:2]),
                 (q, k[:, :1], k[:, :1], pos, freq, slots)):
        with pytest.raises(ValueError):
            kv.norm_rope_append(0, *args)
    with pytest.raises(GGError):
        kv.norm_rope_append(1, q, k, k, pos, freq, slots)
    # No rows: nothing to do, nothing refused.
    assert kv.norm_rope_append(0, q[:0], k[:0], k[:0], pos[:0], freq, slots[:0]).shape == (0, hq, d)
    kv.close()


@pytest.mark.parametrize("d", [128, 66])
def test_norm_of_rows_with_tiny_squares(gv, d):
    """Squares below the normal range: fp32 keeps x^2 = 1e-40 to 2^-150 (7e-6 of it), so the norm, its
    root, to 4e-6, and the rounding of the products adds 2^-22."""
    rng = np.random.default_rng(12)
    x = (1e-20 * rng.uniform(1, 2, (7, 2, d)) * rng.choice([-1, 1], (7, 2, d))).astype(np.float32)
    x[3] = 0
    zero, freq = torch.zeros(7, dtype=torch.int32, device="cuda"), torch.ones(d // 2, device="cuda")
    one = torch.ones(d, device="cuda")
    live = [0, 1, 2, 4, 5, 6]
    got = gv.qk_norm_rope(torch.from_numpy(x).cuda(), None, zero, freq, one, eps=0.0)[0].cpu().numpy()
    want = x.astype(np.float64)[live] / np.sqrt((x.astype(np.float64)[live] ** 2).mean(-1, keepdims=True))
    assert (np.abs(got[live] - want) <= 1e-5 * np.abs(want)).all()
    got = gv.qk_norm_rope(torch.from_numpy(x).cuda(), None, zero, freq, one, eps=1e-6)[0].cpu().numpy()
    assert (np.abs(got - x.astype(np.float64) * 1e3) <= 2.0 ** -21 * np.abs(x) * 1e3).all()


def test_tensors_of_another_device_are_refused(gv, monkeypatch):
    """The current device, as the calls see it, is one that holds none of the tensors."""
    n, hq, h, d = 4, 4, 2, 64
    q, k = torch.zeros(n, hq, d, device="cuda"), torch.zeros(n, h, d, device="cuda")
    pos, freq = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda")
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    kv = gv.KVCache(1, 2, 16, h, d, DType.INT4)
    out = (torch.zeros(n, h, d, device="cuda"), None)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "current_device", lambda: 1)
        for call in (lambda: gv.qk_norm_rope(q, k, pos, freq), lambda: kv.norm_rope_append(0, q, k, k, pos, freq, slots),
                     lambda: kv.read(0, slots, out=out)):
            with pytest.raises(ValueError, match="another device"):
                call()
    kv.close()


def test_axes_of_pairs_in_any_form(gv):
    """Bytes, lists, arrays and tensors of whole numbers name the same axes; anything else is refused."""
    rng = np.random.default_rng(11)
    n, d = 5, 64
    q = torch.from_numpy(rng.normal(0, 1, (n, 2, d)).astype(np.float32)).cuda()
    pos = torch.from_numpy(rng.integers(0, 1000, (2, n)).astype(np.int32)).cuda()
    freq = torch.from_numpy(np.exp2(-rng.uniform(0, 10, 32)).astype(np.float32)).cuda()
    axes = [int(x) for x in rng.integers(0, 2, 32)]
    want = gv.qk_norm_rope(q, None, pos, freq, pair_axis=axes)[0]
    for form in (bytes(axes), tuple(axes), np.array(axes), np.array(axes, dtype=np.uint8), torch.tensor(axes)):
        assert torch.equal(gv.qk_norm_rope(q, None, pos, freq, pair_axis=form)[0], want)
    for bad in (32, np.array(axes) / 2, [300] * 32):
        with pytest.raises((ValueError, TypeError)):
            gv.qk_norm_rope(q, None, pos, freq, pair_axis=bad)


def test_graph_of_a_layer(gv):
    """Norm, rotation and append into the pool, plan and attention: captured once, replayed."""
    rng = np.random.default_rng(6)
    B, R, hq, h, d = 2, 3, 8, 2, 128
    keys = [200, 70]
    kv = gv.KVCache(1, 40, 16, h, d, DType.INT4)
    fill = torch.from_numpy(rng.normal(0, 1, (640, h, d)).astype(np.float32)).cuda()
    kv.append(0, fill, fill.flip(0).contiguous(), torch.arange(640, dtype=torch.int32, device="cuda"))
    tables = torch.arange(26, dtype=torch.int32, device="cuda").view(2, 13).contiguous()
    fused = torch.zeros(B * R, hq + 2 * h, d, dtype=torch.bfloat16, device="cuda")
    pos_np = np.concatenate([np.arange(c - R, c) for c in keys]).astype(np.int32)
    pos = torch.from_numpy(pos_np).cuda()
    slots = torch.from_numpy(np.concatenate([(13 * b + p // 16) * 16 + p % 16 for b, p in enumerate(pos_np.reshape(B, R))]).astype(
        np.int32)).cuda()
    freq = torch.from_numpy((10000.0 ** (-np.arange(64) / 64)).astype(np.float32)).cuda()
    wq, wk = (torch.ones(d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cd = torch.tensor(keys, dtype=torch.int32).cuda()
    ws = kv.attention_workspace(B, R, hq, 13)

    def layer(q_out, out):
        kv.norm_rope_append(0, fused[:, :hq], fused[:, hq:hq + h], fused[:, hq + h:], pos, freq, slots, wq, wk, q_out=q_out)
        kv.attention_plan(cd, R, hq, 13, ws)
        kv.attention(0, q_out.view(B, R, hq, d), out, cd, tables, 0.088, workspace=ws, planned=True)

    q_out = torch.zeros(B * R, hq, d, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(B, R, hq, d, dtype=torch.bfloat16, device="cuda")
    layer(q_out, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        layer(q_out, out)
    for _ in range(4):
        fused.copy_(torch.from_numpy(rng.normal(0, 1, tuple(fused.shape)).astype(np.float32)))
        g.replay()
        got = out.clone()
        e_q, e_o = torch.zeros_like(q_out), torch.zeros_like(out)
        layer(e_q, e_o)
        torch.cuda.synchronize()
        assert torch.equal(got, e_o) and e_o.abs().sum() > 0
    kv.close()


def test_offsets_past_32_bits(gv):
    """Rows 2^20 elements apart: the last ones start past 2^32 bytes."""
    rng = np.random.default_rng(7)
    n, hq, hk, d = 2500, 4, 2, 128
    wide = torch.empty(n, 1 << 20, dtype=torch.bfloat16, device="cuda")
    fused, w, pos, freq, axis = inputs(rng, n, hq, hk, d, "bf16", 64, 1, 5)
    wide[:, :(hq + 2 * hk) * d] = fused.view(n, -1)
    x = wide[:, :(hq + 2 * hk) * d].unflatten(1, (hq + 2 * hk, d))
    kw = dict(positions=torch.from_numpy(pos).cuda(), inv_freq=torch.from_numpy(freq).cuda(), q_weight=w[0], k_weight=w[1])
    a = gv.qk_norm_rope(fused[:, :hq], fused[:, hq:hq + hk], **kw)
    b = gv.qk_norm_rope(x[:, :hq], x[:, hq:hq + hk], **kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    got = []
    for src in (fused, x):
        kv = gv.KVCache(1, n // 16 + 1, 16, hk, d, DType.INT4)
        kv.norm_rope_append(0, src[:, :hq], src[:, hq:hq + hk], src[:, hq + hk:], slot_mapping=slots, **kw)
        got.append(kv.read(0, slots))
        kv.close()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
