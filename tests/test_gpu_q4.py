"""4-bit rows on the GPU: writing and reading back, the score scan, attention, and the engine built of them, against
the definition in 64 bits (tests/q4_util.py).  Tolerances are derived there."""
import math

import numpy as np
import pytest
import torch

from tests import q4_util, util

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _engine(B, H, G, D, rows, dtype="bf16", **kw):
    from diffcache_b200 import DiffCacheGPU

    return DiffCacheGPU(B, H * G, H, D, max_ctx_len=rows, dtype=dtype, store_bits=4, **kw)


def _rows(shape, dtype, seed, spread=True):
    """Normal rows whose 32-element groups span several magnitudes."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    if spread:
        g = torch.randn(shape[:-1] + (shape[-1] // 32, 1), generator=gen)
        x = (x.unflatten(-1, (-1, 32)) * torch.exp(0.7 * g)).flatten(-2)
    return x.to(DTYPES[dtype])


def _nasty_rows(n, D, dtype, seed):
    """Rows where the format is at its edges: ties, zeros, one element only, subnormals, the largest values, NaN, inf."""
    dt, gen = DTYPES[dtype], torch.Generator().manual_seed(seed)
    tiny, big = torch.finfo(dt).tiny, torch.finfo(dt).max
    rows = torch.zeros(n, D, dtype=torch.float64)
    for i in range(n):
        kind = i % 12
        r = torch.randn(D, generator=gen, dtype=torch.float64)
        if kind == 0:      # integers and half-integers with scale exactly 1: every odd half is a tie
            r = torch.randint(-13, 14, (D,), generator=gen).double() / 2
            r[::32] = 7.0
        elif kind == 1:
            r = torch.randint(-13, 14, (D,), generator=gen).double() / 2 * 2.0 ** -9
            r[::32] = -7.0 * 2.0 ** -9
        elif kind == 2:
            r *= 0.0
        elif kind == 3:
            r *= 0.0
            r[i % D] = -3.0
        elif kind == 4:
            r *= tiny * 4
        elif kind == 5:
            r *= tiny / 8
        elif kind == 6:
            r = torch.sign(r) * big
        elif kind == 7:
            r = r / r.abs().max() * big
        elif kind == 8:
            r[5] = math.nan
        elif kind == 9:
            r[D - 1] = -math.inf
        elif kind == 10:
            r = torch.randint(0, 2 ** 15, (D,), generator=gen).double() * 2.0 ** -24   # fp16 subnormals and their neighbours
        rows[i] = r
    return rows.to(dt)


# ---- writing and reading back ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,D,n", [(1, 1, 64, 1), (2, 3, 64, 37), (1, 2, 128, 1), (2, 2, 128, 129), (1, 5, 256, 33), (3, 1, 256, 8)])
def test_write_and_read_back(B, H, D, n, dtype):
    x, y = _rows((B, H, n, D), dtype, 1), _rows((B, H, n, D), dtype, 2)
    eng = _engine(B, H, 1, D, n + 5, dtype)
    eng.prefill(x.cuda(), y.cuda())
    assert eng.ctx_len == n
    k, v = torch.full((B, H, n + 5, D), 9.0, dtype=x.dtype, device="cuda"), torch.full((B, H, n + 5, D), 9.0, dtype=x.dtype, device="cuda")
    eng.read_rows(k, v)
    for got, src in ((k, x), (v, y)):
        assert bit_rows(got[:, :, :n], q4_util.stored(src).to(src.dtype))
        assert (got[:, :, n:] == 0).all()      # rows that are not stored
    keys = torch.from_numpy(eng.get_keys())
    assert torch.equal(keys, q4_util.stored(x).float())


def bit_rows(got, want):
    return q4_util.bit_equal(got.cpu(), want.cpu())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_edges_of_the_format(D, dtype):
    x = _nasty_rows(72, D, dtype, 5).reshape(1, 1, 72, D)
    y = _nasty_rows(73, D, dtype, 6)[1:].reshape(1, 1, 72, D)
    eng = _engine(1, 1, 1, D, 72, dtype)
    eng.prefill(x.cuda(), y.cuda())
    k, v = torch.empty_like(x, device="cuda"), torch.empty_like(x, device="cuda")
    eng.read_rows(k, v)
    for got, src in ((k, x), (v, y)):
        assert bit_rows(got, q4_util.stored(src).to(src.dtype))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_every_value_against_one_scale(dtype):
    """All finite 16-bit patterns below the group's largest element, for scales of several roundings."""
    dt, D = DTYPES[dtype], 128
    bits = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16).view(dt)
    groups = []
    for top in (7.0, 6.9, 1.0, 0.37, 3.3e-5, 123.0):
        vals = bits[torch.isfinite(bits) & (bits.abs() <= torch.tensor(top).to(dt).abs())]
        pad = (-len(vals)) % 31
        vals = torch.cat([vals, vals.new_zeros(pad)]).reshape(-1, 31)
        groups.append(torch.cat([torch.full((len(vals), 1), top).to(dt), vals], 1))
    g = torch.cat(groups)
    g = torch.cat([g, g.new_zeros((-len(g)) % 4, 32)])
    x = g.reshape(1, 1, -1, D)
    eng = _engine(1, 1, 1, D, x.shape[2], dtype)
    eng.prefill(x.cuda(), x.cuda())
    k = torch.empty_like(x, device="cuda")
    eng.read_rows(k, None)
    assert bit_rows(k, q4_util.stored(x).to(dt))


@pytest.mark.parametrize("layout", ["heads_last", "padded", "sliced", "expanded", "host", "host_numpy"])
def test_write_strides_and_chunks(layout):
    """Chunks at odd positions from differently laid out sources; rows outside a chunk keep their contents."""
    B, H, D, n = 2, 3, 128, 50
    x, y = _rows((B, H, n, D), "bf16", 7), _rows((B, H, n, D), "bf16", 8)
    eng = _engine(B, H, 2, D, 64)

    def lay(t):
        if layout == "heads_last":
            return t.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)
        if layout == "padded":
            buf = torch.zeros(B, H + 1, t.shape[2] + 3, D + 8, dtype=t.dtype, device="cuda")
            buf[:, 1:, 2:2 + t.shape[2], :D] = t.cuda()
            return buf[:, 1:, 2:2 + t.shape[2], :D]
        if layout == "sliced":
            return torch.stack([t, t + 1], 3).cuda()[:, :, :, 0]
        if layout == "expanded":
            return t[:1].cuda().expand(B, H, -1, D)
        if layout == "host":
            return t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        return util.u16(t)

    if layout == "expanded":
        x, y = x[:1].expand(B, H, n, D), y[:1].expand(B, H, n, D)
    for lo, hi in ((0, 1), (1, 18), (18, 50), (7, 9)):
        eng.write_rows(lo, lay(x[:, :, lo:hi]), lay(y[:, :, lo:hi]))
        assert eng.ctx_len == max(hi, 50 if (lo, hi) == (7, 9) else hi)
    k, v = torch.empty(B, H, n, D, dtype=x.dtype, device="cuda"), torch.empty(B, H, n, D, dtype=x.dtype, device="cuda")
    eng.read_rows(k, v)
    assert bit_rows(k, q4_util.stored(x).to(x.dtype)) and bit_rows(v, q4_util.stored(y).to(x.dtype))


def test_write_rows_on_a_16_bit_store():
    from diffcache_b200 import DiffCacheGPU

    x, y = _rows((2, 2, 40, 64), "bf16", 9), _rows((2, 2, 40, 64), "bf16", 10)
    eng = DiffCacheGPU(2, 4, 2, 64, max_ctx_len=48)
    for lo, hi in ((0, 17), (17, 40), (3, 5)):
        eng.write_rows(lo, x[:, :, lo:hi].cuda(), y[:, :, lo:hi].cuda())
    k, v = torch.empty(2, 2, 44, 64, dtype=x.dtype, device="cuda"), torch.empty(2, 2, 44, 64, dtype=x.dtype, device="cuda")
    eng.read_rows(k, v, row0=4)
    assert torch.equal(k[:, :, :36].cpu(), x[:, :, 4:]) and torch.equal(v[:, :, :36].cpu(), y[:, :, 4:]) and (k[:, :, 36:] == 0).all()
    ids = torch.tensor([[[3, -1, 39], [0, 40, 3]], [[1, 1, 47], [2, 0, 5]]], dtype=torch.int32).cuda()
    out = torch.empty(2, 2, 3, 64, dtype=x.dtype, device="cuda")
    eng.read_rows(out, None, ids=ids)
    assert torch.equal(out.cpu(), _take(x, ids.cpu(), 40))
    bits = torch.zeros(2, 2, 40, dtype=torch.int32, device="cuda")
    q = _rows((2, 2, 64), "bf16", 11)
    eng.score_rows(q.cuda(), bits)
    dist, tol = q4_util.scan(x.double().reshape(4, 40, 64), q.reshape(4, 64))
    q4_util.assert_close(bits.view(torch.float32).cpu().reshape(4, 40), dist, tol, "dist")


def _take(x, ids, n):
    B, H, _, D = x.shape
    out = torch.zeros(*ids.shape, D, dtype=x.dtype)
    for b in range(B):
        for h in range(H):
            for i, r in enumerate(ids[b, h].tolist()):
                if 0 <= r < n:
                    out[b, h, i] = x[b, h, r]
    return out


@pytest.mark.parametrize("D", [64, 128, 256])
def test_read_by_ids(D):
    B, H, n = 2, 2, 100
    x, y = _rows((B, H, n, D), "fp16", 12), _rows((B, H, n, D), "fp16", 13)
    eng = _engine(B, H, 1, D, 128, "fp16")
    eng.prefill(x.cuda(), y.cuda())
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, n, (B, H, 41), generator=gen, dtype=torch.int32)
    ids[:, :, 3], ids[:, :, 7], ids[:, :, 9], ids[:, :, 11] = -1, n, 127, ids[:, :, 12]
    k, v = torch.full((B, H, 41, D), 5.0, dtype=x.dtype, device="cuda"), torch.full((B, H, 41, D), 5.0, dtype=x.dtype, device="cuda")
    eng.read_rows(k, v, ids=ids.cuda())
    for got, src in ((k, x), (v, y)):
        assert bit_rows(got, _take(q4_util.stored(src).to(src.dtype), ids, n))


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp16", 64), ("bf16", 256)])
def test_insert_appends_what_write_would(dtype, D):
    B, H, n = 2, 3, 21
    x, y = _rows((B, H, n, D), dtype, 14), _rows((B, H, n, D), dtype, 15)
    eng = _engine(B, H, 1, D, n, dtype)
    eng.prefill(x[:, :, :15].cuda(), y[:, :, :15].cuda())
    for i in range(15, n):
        host = i % 2 == 0
        kk, vv = x[:, :, i].contiguous(), y[:, :, i].contiguous()
        eng.insert(util.u16(kk) if host else kk.cuda(), util.u16(vv) if host else vv.cuda())
    assert eng.ctx_len == n
    k, v = torch.empty(B, H, n, D, dtype=x.dtype, device="cuda"), torch.empty(B, H, n, D, dtype=x.dtype, device="cuda")
    eng.read_rows(k, v)
    assert bit_rows(k, q4_util.stored(x).to(x.dtype)) and bit_rows(v, q4_util.stored(y).to(x.dtype))
    from diffcache_b200 import DiffCacheError

    with pytest.raises(DiffCacheError, match="full"):
        eng.insert(x[:, :, 0].contiguous().cuda(), y[:, :, 0].contiguous().cuda())


# ---- scan -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,G,D,n", [(1, 1, 1, 64, 1), (2, 3, 4, 64, 517), (1, 2, 7, 128, 15), (1, 8, 4, 128, 2049), (2, 1, 8, 128, 300),
                                       (1, 2, 3, 256, 1000), (1, 1, 1, 256, 17)])
def test_score_rows(B, H, G, D, n, dtype):
    x = _rows((B, H, n, D), dtype, 20)
    q = _rows((B, H * G, D), dtype, 21, spread=False)
    mean = q.reshape(B, H, G, D).float().mean(2).to(q.dtype)
    eng = _engine(B, H, G, D, n + 3, dtype)
    eng.prefill(x.cuda(), x.cuda())
    bits = torch.full((B, H, n + 2), 77, dtype=torch.int32, device="cuda")
    eng.score_rows(mean.cuda(), bits)
    assert (bits[:, :, n:] == 77).all()       # beyond the stored rows: left as they were
    dist, tol = q4_util.scan(q4_util.stored(x).reshape(B * H, n, D), mean.reshape(B * H, D))
    q4_util.assert_close(bits[:, :, :n].reshape(B * H, n).cpu().view(torch.float32), dist, tol, "dist")
    if G in (1, 4, 8):       # the group mean of two-power groups has one rounding whichever way it is summed
        both = torch.empty(B, H, n, dtype=torch.int32, device="cuda")
        eng.score_rows(q.cuda(), both)
        m64 = q.reshape(B, H, G, D).double().mean(2)
        off = torch.matmul(q4_util.stored(x).reshape(B * H, n, D).abs(),
                           (m64.abs() * q4_util.HALF_STEP[q.dtype] + 2.0 ** -25).reshape(B * H, D, 1)).squeeze(-1)
        dist, tol = q4_util.scan(q4_util.stored(x).reshape(B * H, n, D), m64.reshape(B * H, D))
        q4_util.assert_close(both.reshape(B * H, n).cpu().view(torch.float32), dist, tol + 1.01 * off, "dist from heads")
    small = torch.full((B, H, max(1, n // 2)), 5, dtype=torch.int32, device="cuda")
    eng.score_rows(mean.cuda(), small)
    assert torch.equal(small, bits[:, :, :max(1, n // 2)])


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** 100])
def test_score_rows_far_magnitudes(scale):
    """Keys tiny and queries huge, and the other way round: the product is ordinary."""
    x, q = _rows((1, 2, 200, 128), "bf16", 22), _rows((1, 2, 128), "bf16", 23, spread=False)
    x, q = (x.double() * scale).to(x.dtype), (q.double() / scale).to(q.dtype)
    eng = _engine(1, 2, 1, 128, 200)
    eng.prefill(x.cuda(), x.cuda())
    bits = torch.empty(1, 2, 200, dtype=torch.int32, device="cuda")
    eng.score_rows(q.cuda(), bits)
    dist, tol = q4_util.scan(q4_util.stored(x).reshape(2, 200, 128), q.reshape(2, 128))
    q4_util.assert_close(bits.cpu().view(torch.float32).reshape(2, 200), dist, tol, "dist")


@pytest.mark.parametrize("scale", [2.0 ** -119, 2.0 ** 115])
def test_scores_and_attention_at_the_ends_of_the_range(scale):
    """Keys near the smallest normal numbers with queries near the largest, and the other way round."""
    x, y, q = _rows((1, 2, 200, 128), "bf16", 24, False), _rows((1, 2, 200, 128), "bf16", 25, False), _rows((1, 8, 128), "bf16", 26, False)
    x, q = (x.double() * scale).to(x.dtype), (q.double() / scale).to(q.dtype)
    eng = _engine(1, 2, 4, 128, 200)
    eng.prefill(x.cuda(), y.cuda())
    one = q[:, ::4].contiguous()
    bits = torch.empty(1, 2, 200, dtype=torch.int32, device="cuda")
    eng.score_rows(one.cuda(), bits)
    ks, vs = q4_util.stored(x), q4_util.stored(y)
    dist, tol = q4_util.scan(ks.reshape(2, 200, 128), one.reshape(2, 128))
    q4_util.assert_close(bits.cpu().view(torch.float32).reshape(2, 200), dist, tol, "dist")
    out, lse = torch.empty_like(q, device="cuda"), torch.empty(1, 8, device="cuda")
    eng.attend_rows(q.cuda(), out, out_lse=lse)
    want, wl, to, tl = q4_util.attend(q.reshape(2, 4, 128), ks[0], vs[0], torch.ones(2, 200, dtype=torch.bool), 128 ** -0.5)
    q4_util.assert_close(out.cpu().reshape(2, 4, 128), want, to, "out")
    q4_util.assert_close(lse.cpu().reshape(2, 4), wl, tl, "lse")


def test_scores_and_attention_where_the_large_channel_does_not_count():
    """Every group has one channel 100 times the rest, which the query ignores: the codes that count are small.  The 32-bit
    sums take codes with an offset of 8 and take it back, so their magnitudes are up to (|c| + 16) |q| s an element, and
    the bound of 2^-22 a step holds for those: 16 |q| s more than where only |c| |q| s are summed."""
    B, H, G, D, n = 1, 2, 4, 128, 300
    x, y, q = _rows((B, H, n, D), "bf16", 27, False), _rows((B, H, n, D), "bf16", 28, False), _rows((B, H * G, D), "bf16", 29, False)
    x[..., ::32] *= 100
    q[..., ::32] = 0
    eng = _engine(B, H, G, D, n)
    eng.prefill(x.cuda(), y.cuda())
    one = q[:, ::G].contiguous()
    bits = torch.empty(B, H, n, dtype=torch.int32, device="cuda")
    eng.score_rows(one.cuda(), bits)
    ks, vs = q4_util.stored(x), q4_util.stored(y)
    steps = q4_util.quantise(x)[1].expand(B, H, n, D // 32, 32).reshape(H, n, D)
    dist, tol = q4_util.scan(ks.reshape(H, n, D), one.reshape(H, D))
    more = 16 * D * 2.0 ** -22 * torch.matmul(steps, one.reshape(H, D, 1).double().abs()).squeeze(-1)
    q4_util.assert_close(bits.cpu().view(torch.float32).reshape(H, n), dist, tol + more, "dist")
    out, lse = torch.empty_like(q, device="cuda"), torch.empty(B, H * G, device="cuda")
    eng.attend_rows(q.cuda(), out, out_lse=lse)
    qh = q.reshape(H, G, D)
    want, wl, to, tl = q4_util.attend(qh, ks[0], vs[0], torch.ones(H, n, dtype=torch.bool), D ** -0.5)
    more = 16 * D * 2.0 ** -22 * D ** -0.5 * torch.matmul(qh.double().abs(), steps.transpose(1, 2)).amax(-1)
    q4_util.assert_close(lse.cpu().reshape(H, G), wl, tl + more, "lse")
    to = to + 2.02 * more.unsqueeze(-1) * vs[0].abs().amax(1, keepdim=True)     # every weight off by that factor, |v| at most its largest
    q4_util.assert_close(out.cpu().reshape(H, G, D), want, to, "out")


# ---- attention ------------------------------------------------------------------------------------------------------

def _attend_case(B, H, G, D, n, dtype, seed, ids=None, lens=None, res=0, new=False, scale=0.0, spread=False, prep=None):
    x, y = _rows((B, H, n, D), dtype, seed, spread), _rows((B, H, n, D), dtype, seed + 1, spread)
    if prep is not None:
        prep(x, y)
    q = _rows((B, H * G, D), dtype, seed + 2, False)
    rk, rv = _rows((B, H, res + 4, D), dtype, seed + 3, False), _rows((B, H, res + 4, D), dtype, seed + 4, False)
    kn, vn = _rows((B, H, D), dtype, seed + 5, False), _rows((B, H, D), dtype, seed + 6, False)
    eng = _engine(B, H, G, D, n + 7, dtype)
    eng.prefill(x.cuda(), y.cuda())
    out = torch.full((B, H * G, D), 3.0, dtype=q.dtype, device="cuda")
    lse = torch.full((B, H * G), 3.0, dtype=torch.float32, device="cuda")
    drk, drv = rk.cuda(), rv.cuda()
    kw = {}
    if res or new:
        kw.update(res_k=drk, res_v=drv, res_len=res)
    if new:
        kw.update(k_new=kn.cuda(), v_new=vn.cuda())
    if ids is not None:
        kw["ids"] = ids.cuda()
    if lens is not None:
        kw["lens"] = lens.cuda()
    eng.attend_rows(q.cuda(), out, out_lse=lse, scale=scale, **kw)
    torch.cuda.synchronize()
    ks, vs = q4_util.stored(x), q4_util.stored(y)
    for b in range(B):
        for h in range(H):
            if ids is not None:
                pick = ids[b, h].long()
                pick = pick[(pick >= 0) & (pick < n)]
                kk, vv = ks[b, h][pick], vs[b, h][pick]
            else:
                m = n if lens is None else max(0, min(n, int(lens[b])))
                kk, vv = ks[b, h, :m], vs[b, h, :m]
            parts_k, parts_v = [kk, rk[b, h, :res].double()], [vv, rv[b, h, :res].double()]
            if new:
                parts_k.append(kn[b, h].double()[None])
                parts_v.append(vn[b, h].double()[None])
            kk, vv = torch.cat(parts_k), torch.cat(parts_v)
            qq = q[b, h * G:(h + 1) * G][None]
            if kk.shape[0] == 0:
                assert (out[b, h * G:(h + 1) * G] == 0).all() and (lse[b, h * G:(h + 1) * G] == -math.inf).all()
                continue
            want, wl, to, tl = q4_util.attend(qq, kk[None], vv[None], torch.ones(1, kk.shape[0], dtype=torch.bool),
                                              scale if scale > 0 else D ** -0.5)
            q4_util.assert_close(out[b, h * G:(h + 1) * G].cpu()[None], want, to, f"out {b},{h}")
            q4_util.assert_close(lse[b, h * G:(h + 1) * G].cpu()[None], wl, tl, f"lse {b},{h}")
    if new:
        assert torch.equal(drk[:, :, res].cpu(), kn) and torch.equal(drv[:, :, res].cpu(), vn)
    keep = res + (1 if new else 0)
    assert torch.equal(drk[:, :, keep:].cpu(), rk[:, :, keep:])
    return eng, out, lse


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,G,D,n", [(1, 1, 1, 64, 1), (2, 2, 4, 64, 130), (1, 2, 8, 128, 65), (1, 8, 4, 128, 1500), (2, 1, 5, 256, 77),
                                       (1, 1, 16, 128, 333), (1, 2, 12, 64, 47), (3, 1, 1, 256, 16), (1, 1, 3, 128, 4099)])
def test_attend_all_rows(B, H, G, D, n, dtype):
    _attend_case(B, H, G, D, n, dtype, 40)


@pytest.mark.parametrize("G,D,res,new", [(4, 128, 0, True), (4, 128, 70, True), (8, 64, 1, False), (1, 256, 33, True), (9, 128, 576, False),
                                         (2, 64, 200, True)])
def test_attend_with_resident_rows_and_new_token(G, D, res, new):
    _attend_case(2, 2, G, D, 90, "bf16", 50, res=res, new=new)
    _attend_case(1, 2, G, D, 90, "fp16", 51, ids=torch.randperm(90)[:64].reshape(1, 2, 32).to(torch.int32), res=res, new=new)


@pytest.mark.parametrize("dtype,G", [("bf16", 4), ("fp16", 8), ("bf16", 1)])
def test_attend_padded_batch(dtype, G):
    """Lengths of zero, one, inside a tile, all rows, beyond the store, negative; one sequence with nothing at all."""
    lens = torch.tensor([0, 1, 15, 16, 17, 200, 1000, -3], dtype=torch.int32)
    _attend_case(8, 2, G, 128, 200, dtype, 60, lens=lens)
    _attend_case(8, 2, G, 64, 200, dtype, 61, lens=lens, res=5, new=True)


@pytest.mark.parametrize("k", [1, 15, 16, 31, 100, 513])
def test_attend_ids(k):
    B, H, n = 2, 2, 700
    gen = torch.Generator().manual_seed(k)
    ids = torch.stack([torch.randperm(n, generator=gen)[:k] for _ in range(B * H)]).reshape(B, H, k).to(torch.int32)
    _attend_case(B, H, 4, 128, n, "bf16", 70, ids=ids)
    if k > 4:
        ids[0, 0, 1], ids[0, 1, k - 1], ids[1, 0, 2], ids[1, 1, 3] = -1, n, ids[1, 0, 0], 2 ** 31 - 1   # pads, ids not stored, a repeat
        _attend_case(B, H, 3, 64, n, "fp16", 71, ids=ids, res=3, new=True)
    none = torch.full((B, H, k), -1, dtype=torch.int32)
    none[0, 0, 0] = 5
    _attend_case(B, H, 4, 128, n, "bf16", 72, ids=none)


def test_attend_no_ids_at_all():
    none = torch.empty((1, 2, 0), dtype=torch.int32)
    _attend_case(1, 2, 4, 128, 30, "bf16", 73, ids=none)
    _attend_case(1, 2, 4, 128, 30, "bf16", 74, ids=none, res=2, new=True)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attend_sharp_and_spread_inputs(dtype):
    """A large softmax scale (one row takes almost everything, the maximum moves) and groups of unequal magnitude."""
    _attend_case(1, 2, 4, 128, 400, dtype, 80, scale=2.0)
    _attend_case(1, 2, 8, 64, 400, dtype, 81, spread=True)
    _attend_case(1, 2, 2, 256, 100, dtype, 82, scale=1e-6, spread=True)


def test_attend_far_value_magnitudes():
    def prep(x, y):
        y *= 2.0 ** 90
        y[:, :, ::3] *= 2.0 ** -80
    _attend_case(1, 2, 4, 128, 300, "bf16", 83, prep=prep)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_bad_rows_matter_only_where_they_are_attended(bad):
    B, H, G, D, n = 2, 2, 4, 128, 64
    def prep(x, y):
        x[:, :, 40:] = bad
        y[:, :, 40:] = -bad
    _attend_case(B, H, G, D, n, "bf16", 84, lens=torch.tensor([40, 3], dtype=torch.int32), prep=prep)
    _attend_case(B, H, G, D, n, "bf16", 85, ids=torch.arange(40).expand(B, H, 40).contiguous().to(torch.int32), prep=prep)
    eng = _engine(B, H, G, D, n)
    x, y, q = _rows((B, H, n, D), "bf16", 86), _rows((B, H, n, D), "bf16", 87), _rows((B, H * G, D), "bf16", 88)
    x[0, 1, 5, 7] = bad
    y[1, 0, 6, 100] = bad
    eng.prefill(x.cuda(), y.cuda())
    out, lse = torch.empty_like(q, device="cuda"), torch.empty(B, H * G, device="cuda")
    eng.attend_rows(q.cuda(), out, out_lse=lse)
    o = torch.isnan(out).cpu().reshape(B, H, G, D)
    assert o[0, 1].all() and not o[0, 0].any() and not o[1, 1].any()
    assert o[1, 0, :, 96:].all() and not o[1, 0, :, :96].any()      # the group of the bad value, no other
    assert torch.isnan(lse[0, G:]).all() and torch.isfinite(lse[1]).all()
    bits = torch.empty(B, H, n, dtype=torch.int32, device="cuda")
    eng.score_rows(q.reshape(B, H, G, D)[:, :, 0].contiguous().cuda(), bits)
    nan = torch.isnan(bits.view(torch.float32)).cpu()
    assert nan[0, 1, 5] and int(nan.sum()) == 1


def test_attend_takes_slices_of_a_projection():
    B, H, G, D, n, res = 3, 2, 4, 128, 50, 6
    x, y = _rows((B, H, n, D), "bf16", 90), _rows((B, H, n, D), "bf16", 91)
    qkv = _rows((B, (H * G + 2 * H) * D), "bf16", 92, False).cuda()
    nq, nk = H * G * D, H * D
    q, kn, vn = qkv[:, :nq].unflatten(1, (H * G, D)), qkv[:, nq:nq + nk].unflatten(1, (H, D)), qkv[:, nq + nk:].unflatten(1, (H, D))
    buf = _rows((2, B, H, 40, D), "bf16", 93, False).cuda()
    eng = _engine(B, H, G, D, n)
    eng.prefill(x.cuda(), y.cuda())
    a, b = torch.empty(B, H * G, D, dtype=x.dtype, device="cuda"), torch.empty(B, H * G, D, dtype=x.dtype, device="cuda")
    v1, v2 = buf.clone(), buf.clone()
    eng.attend_rows(q, a, res_k=v1[0][:, :, 30:], res_v=v1[1][:, :, 30:], res_len=res, k_new=kn, v_new=vn)
    eng.attend_rows(q.contiguous(), b, res_k=v2[0][:, :, 30:].contiguous(), res_v=v2[1][:, :, 30:].contiguous(), res_len=res,
                    k_new=kn.contiguous(), v_new=vn.contiguous())
    assert torch.equal(a, b)
    assert torch.equal(v1[0][:, :, 30 + res], kn) and torch.equal(v1[:, :, :, :30 + res], buf[:, :, :, :30 + res])


def test_attend_rows_on_a_16_bit_store_takes_ids_only():
    from diffcache_b200 import DiffCacheGPU

    B, H, G, D, n = 1, 2, 4, 128, 60
    x, y, q = _rows((B, H, n, D), "bf16", 94), _rows((B, H, n, D), "bf16", 95), _rows((B, H * G, D), "bf16", 96, False)
    eng = DiffCacheGPU(B, H * G, H, D, max_ctx_len=n)
    eng.prefill(x.cuda(), y.cuda())
    ids = torch.arange(0, 60, 3, dtype=torch.int32).expand(B, H, 20).contiguous()
    out = torch.empty_like(q, device="cuda")
    eng.attend_rows(q.cuda(), out, ids=ids.cuda())
    want, _, tol, _ = q4_util.attend(q.reshape(H, G, D), x[0, :, ::3].double(), y[0, :, ::3].double(),
                                     torch.ones(H, 20, dtype=torch.bool), D ** -0.5)
    q4_util.assert_close(out.cpu().reshape(H, G, D), want, tol, "out")
    with pytest.raises(ValueError, match="store_bits=4"):
        eng.attend_rows(q.cuda(), out)


# ---- the engine ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("B,H,G,D,n,topk,res,dtype", [(2, 2, 4, 128, 3000, 256, 40, "bf16"), (1, 3, 2, 64, 500, 500, 7, "fp16"),
                                                      (1, 2, 8, 256, 900, 64, 0, "bf16"), (1, 1, 4, 128, 40, 64, 3, "fp16")])
def test_fused_decode_step(B, H, G, D, n, topk, res, dtype):
    """Scan, select and attention together, as a decode step runs them."""
    x, y = _rows((B, H, n, D), dtype, 100, False), _rows((B, H, n, D), dtype, 101, False)
    q = _rows((B, H * G, D), dtype, 102, False)
    rk, rv = _rows((B, H, res + 2, D), dtype, 103, False), _rows((B, H, res + 2, D), dtype, 104, False)
    kn, vn = _rows((B, H, D), dtype, 105, False), _rows((B, H, D), dtype, 106, False)
    eng = _engine(B, H, G, D, n, dtype)
    eng.prefill(x.cuda(), y.cuda())
    k = min(topk, n)
    out, idx = torch.empty_like(q, device="cuda"), torch.empty(B, H, k, dtype=torch.int32, device="cuda")
    lse = torch.empty(B, H * G, device="cuda")
    drk, drv = rk.cuda(), rv.cuda()
    eng.decode_attend(q.cuda(), out, topk, res_k=drk, res_v=drv, res_len=res, k_new=kn.cuda(), v_new=vn.cuda(), out_idx=idx, out_lse=lse)
    eng.check_status()
    bits = torch.empty(B, H, n, dtype=torch.int32, device="cuda")
    eng.score_rows(q.cuda(), bits)
    # the rows chosen are the k smallest ranking keys, ties to the smaller id
    order = np.argsort(bits.cpu().numpy().view(np.uint32).astype(np.uint64) * 2 ** 32 + np.arange(n, dtype=np.uint64), axis=-1, kind="stable")
    assert np.array_equal(idx.cpu().numpy(), order[..., :k].astype(np.int32))
    ks, vs = q4_util.stored(x), q4_util.stored(y)
    for b in range(B):
        for h in range(H):
            pick = idx[b, h].cpu().long()
            kk = torch.cat([ks[b, h][pick], rk[b, h, :res].double(), kn[b, h].double()[None]])
            vv = torch.cat([vs[b, h][pick], rv[b, h, :res].double(), vn[b, h].double()[None]])
            want, wl, to, tl = q4_util.attend(q[b, h * G:(h + 1) * G][None], kk[None], vv[None],
                                              torch.ones(1, kk.shape[0], dtype=torch.bool), D ** -0.5)
            q4_util.assert_close(out[b, h * G:(h + 1) * G].cpu()[None], want, to, "out")
            q4_util.assert_close(lse[b, h * G:(h + 1) * G].cpu()[None], wl, tl, "lse")
    assert torch.equal(drk[:, :, res].cpu(), kn)
    again = torch.empty_like(out)
    eng.attend_rows(q.cuda(), again, ids=idx, res_k=drk, res_v=drv, res_len=res, k_new=kn.cuda(), v_new=vn.cuda())
    assert torch.equal(again, out)


def test_query_returns_the_rows_read_back():
    B, H, D, n, ef = 2, 2, 128, 400, 50
    x, y = _rows((B, H, n, D), "bf16", 110), _rows((B, H, n, D), "bf16", 111)
    q = _rows((B, H, D), "bf16", 112, False)
    eng = _engine(B, H, 4, D, n)
    eng.prefill(util.u16(x), util.u16(y))     # host rows
    kk, vv = np.empty((B, H, ef, D), np.uint16), np.empty((B, H, ef, D), np.uint16)
    idx = np.empty((B, H, ef), np.int32)
    eng.query(kk, vv, util.u16(q), ef, out_idx=idx)
    ids = torch.from_numpy(idx)
    for got, src in ((kk, x), (vv, y)):
        assert bit_rows(torch.from_numpy(got).view(torch.bfloat16), _take(q4_util.stored(src).to(src.dtype), ids, n))


def test_snapshot_round_trip(tmp_path):
    B, H, D, n = 2, 2, 64, 33
    x, y = _rows((B, H, n, D), "fp16", 113), _rows((B, H, n, D), "fp16", 114)
    a, b = _engine(B, H, 1, D, 40, "fp16"), _engine(B, H, 1, D, 50, "fp16")
    a.prefill(x.cuda(), y.cuda())
    a.save(str(tmp_path / "snap_"))
    b.load(str(tmp_path / "snap_"), 40)
    assert b.ctx_len == n
    out = [torch.empty(B, H, n, D, dtype=x.dtype, device="cuda") for _ in range(4)]
    a.read_rows(out[0], out[1])
    b.read_rows(out[2], out[3])
    assert torch.equal(out[0], out[2]) and torch.equal(out[1], out[3])
    from diffcache_b200 import DiffCacheGPU

    c = DiffCacheGPU(B, H, H, D, max_ctx_len=40, dtype="fp16")
    with pytest.raises(ValueError, match="store_bits=4"):
        c.load(str(tmp_path / "snap_"), 40)
    c.prefill(x.cuda(), y.cuda())
    c.save(str(tmp_path / "wide_"))
    b.load(str(tmp_path / "wide_"), 40)       # 16-bit rows, quantised on the way in
    b.read_rows(out[2], out[3])
    assert torch.equal(out[0], out[2]) and torch.equal(out[1], out[3])


def test_sharded_halves_equal_one_engine():
    """Two engines holding the two halves of the rows, merged, against one engine on all rows (emulated on one GPU)."""
    from diffcache_b200 import _lib

    lib = _lib.load()
    B, H, G, D, n, k = 1, 2, 4, 128, 1000, 64
    x, y, q = _rows((B, H, n, D), "bf16", 115), _rows((B, H, n, D), "bf16", 116), _rows((B, H * G, D), "bf16", 117, False).cuda()
    P = B * H
    whole = _engine(B, H, G, D, n)
    whole.prefill(x.cuda(), y.cuda())
    want, idx = torch.empty_like(q), torch.empty(B, H, k, dtype=torch.int32, device="cuda")
    whole.decode_attend(q, want, k, out_idx=idx)
    parts = [_engine(B, H, G, D, n // 2) for _ in range(2)]
    bits = torch.empty(2, P, k, dtype=torch.int32, device="cuda")
    gidx = torch.empty(2, P, k, dtype=torch.int32, device="cuda")
    acc, ml = torch.empty(2, B, H * G, D, device="cuda"), torch.empty(2, B, H * G, 2, device="cuda")
    for r, e in enumerate(parts):
        lo = r * (n // 2)
        e.prefill(x[:, :, lo:lo + n // 2].cuda(), y[:, :, lo:lo + n // 2].cuda())
        e.set_row_offset(lo)
        e.local_topk(q, k, bits[r], gidx[r])
    for r, e in enumerate(parts):
        count = torch.empty(P, dtype=torch.int32, device="cuda")
        _lib.check(lib.dc_merge_sorted_count(bits.data_ptr(), 2, P, k, r, count.data_ptr(), 0))
        torch.cuda.synchronize()
        e.attend_owned(q, gidx[r], k, acc[r], ml[r], sel_count=count)
    out = torch.empty_like(q)
    _lib.check(lib.dc_lse_combine(acc.data_ptr(), acc.stride(0), ml.data_ptr(), ml.stride(0), 2, B * H * G, D, 0, out.data_ptr(),
                                  None, int(torch.cuda.current_stream().cuda_stream)))
    # the same rows in other sums: both are within the 64-bit tolerance, so twice that apart at most
    ks, vs = q4_util.stored(x)[0], q4_util.stored(y)[0]
    pick = idx[0].cpu().long()
    ref, _, tol, _ = q4_util.attend(q.cpu().reshape(H, G, D), torch.stack([ks[h][pick[h]] for h in range(H)]),
                                    torch.stack([vs[h][pick[h]] for h in range(H)]), torch.ones(H, k, dtype=torch.bool), D ** -0.5)
    q4_util.assert_close(out.cpu().reshape(H, G, D), ref, tol, "merged")
    q4_util.assert_close(want.cpu().reshape(H, G, D), ref, tol, "whole")


@pytest.mark.parametrize("n,topk,world", [(1500, 64, 2), (7, 16, 3)])
def test_sequence_sharded_step_over_peer_stores(n, topk, world):
    """The sequence-sharded step on 4-bit engines with both exchanges done by the step's kernels, all ranks emulated on this
    GPU phase by phase (the small case leaves ranks with a few rows and pads)."""
    import ctypes

    from diffcache_b200 import sharded

    B, H, G, D, res = 1, 2, 4, 128, 9
    x, y, q = _rows((B, H, n, D), "bf16", 230), _rows((B, H, n, D), "bf16", 231), _rows((B, H * G, D), "bf16", 232, False)
    rk, rv = _rows((B, H, res + 2, D), "bf16", 233, False), _rows((B, H, res + 2, D), "bf16", 234, False)
    kn, vn = _rows((B, H, D), "bf16", 235, False), _rows((B, H, D), "bf16", 236, False)
    engines, backends = [], []
    for r, (start, length) in enumerate(sharded.shard_rows(n, world)):
        e = _engine(B, H, G, D, max(length, 1))
        if length:
            e.prefill(x[:, :, start:start + length].contiguous().cuda(), y[:, :, start:start + length].contiguous().cuda())
        last = r == world - 1
        engines.append(e)
        backends.append(sharded.GpuShardBackend(e, start, rk.cuda() if last else None, rv.cuda() if last else None, res if last else 0,
                                                kn.cuda() if last else None, vn.cuda() if last else None))
    need = (ctypes.c_int64 * 2)()
    assert backends[0].lib.dc_sharded_slot_bytes(engines[0]._h, topk, need) == 0
    xs = sharded.PeerExchange.in_process([int(need[0]), int(need[1])], [torch.cuda.current_device()] * world)
    qd = q.cuda()
    for _ in range(2):
        for phase in range(3):
            outs = [b.peer_phase(phase, qd, topk, z) for b, z in zip(backends, xs)]
        torch.cuda.synchronize()
    assert all(torch.equal(o, outs[0]) for o in outs)
    for z in xs:
        z.check()
        z.close()
    whole = _engine(B, H, G, D, n)
    whole.prefill(x.cuda(), y.cuda())
    k = min(topk, n)
    one, idx = torch.empty_like(qd), torch.empty(B, H, k, dtype=torch.int32, device="cuda")
    whole.decode_attend(qd, one, topk, res_k=rk.cuda(), res_v=rv.cuda(), res_len=res, k_new=kn.cuda(), v_new=vn.cuda(), out_idx=idx)
    ks, vs = q4_util.stored(x), q4_util.stored(y)
    for h in range(H):
        pick = idx[0, h].cpu().long()
        kk = torch.cat([ks[0, h][pick], rk[0, h, :res].double(), kn[0, h].double()[None]])
        vv = torch.cat([vs[0, h][pick], rv[0, h, :res].double(), vn[0, h].double()[None]])
        want, _, tol, _ = q4_util.attend(q[0, h * G:(h + 1) * G][None], kk[None], vv[None], torch.ones(1, len(kk), dtype=torch.bool),
                                         D ** -0.5)
        q4_util.assert_close(outs[0].reshape(H, G, D)[h].cpu()[None], want, tol, f"sharded {h}")
        q4_util.assert_close(one[0, h * G:(h + 1) * G].cpu()[None], want, tol, f"whole {h}")


def test_kv_cache_manager_prefill_cache_round_trip(tmp_path):
    from diffcache_b200 import DiffCache

    L, B, H, G, D, S = 2, 2, 2, 4, 64, 300
    kw = dict(num_layers=L, batch_size=B, max_length=S + 32, num_kv_heads=H, num_q_heads=H * G, head_dim=D, retrieval_budget=64,
              kvbuf_prefix_len=16, kvbuf_suffix_len=24, kvbuf_suffix_maxlen=48, store_bits=4)
    a = DiffCache(**kw)
    for l in range(L):
        a.prefill_update_kv_cache(_rows((B, S, H, D), "bf16", 240 + l, False).cuda(), _rows((B, S, H, D), "bf16", 250 + l, False).cuda(), l)
    (tmp_path / "cache").mkdir()
    a.save_prefill_cache(str(tmp_path / "cache"))
    b = DiffCache(**kw)
    b.load_prefill_cache(torch.zeros((B, S), dtype=torch.long), str(tmp_path / "cache"))
    for l in range(L):
        q, kn, vn = (_rows((B, 1, h * D), "bf16", 260 + h, False).cuda() for h in (H * G, H, H))
        ia, ib = torch.zeros((B, H, 64), dtype=torch.int32, device="cuda"), torch.zeros((B, H, 64), dtype=torch.int32, device="cuda")
        oa = a.decode_attention(l, q, kn.view(B, 1, H, D), vn.view(B, 1, H, D), out_idx=ia)
        ob = b.decode_attention(l, q, kn.view(B, 1, H, D), vn.view(B, 1, H, D), out_idx=ib)
        assert torch.equal(ia, ib) and torch.equal(oa, ob)
    # the reference's three-call shape: the retrieved rows arrive in the element type
    c = DiffCache(**kw)
    k, v = _rows((B, S, H, D), "bf16", 240, False), _rows((B, S, H, D), "bf16", 250, False)
    c.prefill_update_kv_cache(k.cuda(), v.cuda(), 0)
    c.decode_pre_query_operation(_rows((B, 1, H * G * D), "bf16", 270, False).cuda())
    c.decode_query_kvcache(0)
    c.decode_post_query_operation(0)
    got = c.get_kvcache(0)[0][:, :64].permute(0, 2, 1, 3).cpu()
    mid = (q4_util.stored(k[:, 16:S - 24].permute(0, 2, 1, 3)) + 0.0).to(torch.bfloat16)   # + 0.0: a zero without sign
    for bb in range(B):
        for h in range(H):
            rows = {tuple(r.tolist()) for r in mid[bb, h].view(torch.int16)}
            assert all(tuple(r.tolist()) in rows for r in got[bb, h].view(torch.int16))


def test_attention_stack_on_4_bit_stores():
    from diffcache_b200.stack import AttentionStack

    B, HQ, H, D, n, topk, sink, win = 2, 8, 2, 128, 700, 96, 16, 32
    st = AttentionStack(2, 256, B, HQ, H, D, n, topk, sink, win, store_bits=4)
    probe = {}
    x = torch.randn(B, 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    out = st.step(x, probe=probe)
    assert torch.isfinite(out).all() and all(e.store_bits == 4 for e in st.engines)
    eng, n_r = st.engines[0], n - sink - win
    idx = torch.empty(B, H, topk, dtype=torch.int32, device="cuda")
    again = torch.empty_like(probe["attn"])
    eng.decode_attend(probe["q"].contiguous(), again, topk, res_k=st.res_k[0], res_v=st.res_v[0], res_len=st.res_rows,
                      k_new=probe["k_new"].contiguous(), v_new=probe["v_new"].contiguous(), out_idx=idx)
    assert torch.equal(again, probe["attn"])
    codes = torch.empty(B, H, n_r, D, dtype=torch.bfloat16, device="cuda"), torch.empty(B, H, n_r, D, dtype=torch.bfloat16, device="cuda")
    eng.read_rows(*codes)        # the stored rows rounded to the element type: within half a step of what is attended
    G = HQ // H
    for b in range(B):
        for h in range(H):
            pick = idx[b, h].cpu().long()
            kk = torch.cat([codes[0][b, h].cpu()[pick], st.res_k[0][b, h, :st.res_rows].cpu(), probe["k_new"][b, h].cpu()[None]]).double()
            vv = torch.cat([codes[1][b, h].cpu()[pick], st.res_v[0][b, h, :st.res_rows].cpu(), probe["v_new"][b, h].cpu()[None]]).double()
            q = probe["q"][b, h * G:(h + 1) * G].cpu()
            want, _, tol, _ = q4_util.attend(q[None], kk[None], vv[None], torch.ones(1, len(kk), dtype=torch.bool), D ** -0.5)
            # every key element off by half a step moves a logit by that part of the magnitudes it sums; values likewise
            mag = (q.double().abs() @ kk.abs().T).amax() * D ** -0.5
            slack = (2 * 2.0 ** -8 * mag + 2.0 ** -8) * vv.abs().amax()
            q4_util.assert_close(probe["attn"][b, h * G:(h + 1) * G].cpu()[None], want, tol + slack, "attn")
    st.close()


def test_decode_loop_with_ring_and_spill_from_one_graph():
    """A KV-cache manager on 4-bit stores: captured decode steps past the full window; spilled tokens land in the store."""
    from diffcache_b200 import DiffCache

    B, H, G, D, n, cap, budget = 2, 2, 4, 64, 120, 6, 48
    cache = DiffCache(1, B, 200, H, H * G, D, budget, kvbuf_prefix_len=4, kvbuf_suffix_len=5, kvbuf_suffix_maxlen=cap, store_bits=4)
    x, y = _rows((B, n, H, D), "bf16", 120, False), _rows((B, n, H, D), "bf16", 121, False)
    cache.prefill_update_kv_cache(x.cuda(), y.cuda(), 0)
    store_k, store_v = list(x[:, 4:n - 5].unbind(1)), list(y[:, 4:n - 5].unbind(1))
    res_k, res_v = list(x[:, :4].unbind(1)) + list(x[:, n - 5:].unbind(1)), list(y[:, :4].unbind(1)) + list(y[:, n - 5:].unbind(1))
    q, kn, vn = (torch.zeros(B, h, D, dtype=torch.bfloat16, device="cuda") for h in (H * G, H, H))
    out = torch.empty_like(q)
    idx = torch.empty(B, H, budget, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    win0 = cache._win.clone()
    buf0 = cache.kbuf[0].clone(), cache.vbuf[0].clone()
    with torch.cuda.stream(stream):
        cache.decode_attention(0, q, kn, vn, out=out, out_idx=idx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        cache.decode_attention(0, q, kn, vn, out=out, out_idx=idx)
    cache._win.copy_(win0)
    cache.kbuf[0].copy_(buf0[0]); cache.vbuf[0].copy_(buf0[1])
    order_k, order_v = res_k[4:], res_v[4:]
    for step in range(10):
        tq, tk, tv = _rows((B, H * G, D), "bf16", 200 + step, False), _rows((B, H, D), "bf16", 300 + step, False), _rows((B, H, D), "bf16", 400 + step, False)
        q.copy_(tq); kn.copy_(tk); vn.copy_(tv)
        graph.replay()
        torch.cuda.synchronize()
        if len(order_k) == cap:
            store_k.append(order_k.pop(0)); store_v.append(order_v.pop(0))
        order_k.append(tk); order_v.append(tv)
        ks, vs = q4_util.stored(torch.stack(store_k, 2)), q4_util.stored(torch.stack(store_v, 2))
        rk, rv = torch.stack(res_k[:4] + order_k, 2).double(), torch.stack(res_v[:4] + order_v, 2).double()
        for b in range(B):
            for h in range(H):
                pick = idx[b, h].cpu().long()
                kk, vv = torch.cat([ks[b, h][pick], rk[b, h]]), torch.cat([vs[b, h][pick], rv[b, h]])
                want, _, tol, _ = q4_util.attend(tq[b, h * G:(h + 1) * G][None], kk[None], vv[None],
                                                 torch.ones(1, kk.shape[0], dtype=torch.bool), D ** -0.5)
                q4_util.assert_close(out[b, h * G:(h + 1) * G].cpu()[None], want, tol, f"step {step}")
    cache.data_layers[0].check_status()
    cache.sync_lengths()
    assert cache.retrieval_region_len == len(store_k)
    k = torch.empty(B, H, len(store_k), D, dtype=torch.bfloat16, device="cuda")
    cache.data_layers[0].read_rows(k, None)
    assert bit_rows(k, q4_util.stored(torch.stack(store_k, 2)).to(torch.bfloat16))
    from diffcache_b200 import DiffCacheError

    with pytest.raises(DiffCacheError, match="only the device knows"):
        cache.data_layers[0].write_rows(0, k, k)


def test_captured_calls_replay_with_new_inputs_on_another_stream():
    B, H, G, D, n = 2, 2, 4, 128, 260
    x, y = _rows((B, H, n, D), "bf16", 130), _rows((B, H, n, D), "bf16", 131)
    eng = _engine(B, H, G, D, 300)
    eng.prefill(x.cuda(), y.cuda())
    q = torch.zeros(B, H * G, D, dtype=torch.bfloat16, device="cuda")
    chunk = torch.zeros(2, B, H, 20, D, dtype=torch.bfloat16, device="cuda")
    out, bits = torch.empty_like(q), torch.empty(B, H, n, dtype=torch.int32, device="cuda")
    back = torch.empty(B, H, 20, D, dtype=torch.bfloat16, device="cuda")
    lens = torch.tensor([n, 9], dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()

    def calls():
        eng.write_rows(100, chunk[0], chunk[1])
        eng.read_rows(back, None, row0=100)
        eng.score_rows(q, bits)
        eng.attend_rows(q, out, lens=lens)

    with torch.cuda.stream(stream):
        calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        calls()
    for i in range(3):
        q.copy_(_rows((B, H * G, D), "bf16", 140 + i, False))
        chunk.copy_(_rows((2, B, H, 20, D), "bf16", 150 + i))
        lens.copy_(torch.tensor([n - 50 * i, 9 + 100 * i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), bits.clone(), back.clone()
        calls()
        torch.cuda.synchronize()
        # eager launches make the same splits of the same rows (the store's bound differs: the sums may not)
        assert torch.equal(got[1], bits) and torch.equal(got[2], back)
        x2, y2 = x.clone(), y.clone()
        x2[:, :, 100:120], y2[:, :, 100:120] = chunk[0].cpu(), chunk[1].cpu()
        for b in range(B):
            m = int(lens[b])
            for h in range(H):
                want, _, tol, _ = q4_util.attend(q[b, h * G:(h + 1) * G].cpu()[None], q4_util.stored(x2[b, h, :m])[None],
                                                 q4_util.stored(y2[b, h, :m])[None], torch.ones(1, m, dtype=torch.bool), D ** -0.5)
                for o in (got[0], out):
                    q4_util.assert_close(o[b, h * G:(h + 1) * G].cpu()[None], want, tol, "out")


def test_stateless_functions_equal_the_engine():
    from diffcache_b200 import _lib

    lib = _lib.load()
    B, H, G, D, n, rows = 2, 2, 4, 128, 150, 170
    P = B * H
    x, y, q = _rows((B, H, n, D), "fp16", 160).cuda(), _rows((B, H, n, D), "fp16", 161).cuda(), _rows((B, H * G, D), "fp16", 162, False).cuda()
    st = int(torch.cuda.current_stream().cuda_stream)
    bufs = [torch.full((P, rows, d), fill, dtype=t, device="cuda") for _ in range(2) for d, t, fill in ((D // 2, torch.uint8, 200), (D // 32, torch.float16, 3.0))]
    _lib.check(lib.dc_q4_write_rows(x.data_ptr(), y.data_ptr(), H * n * D, n * D, D, P, H, n, D, 1, *(t.data_ptr() for t in bufs), rows, 11, st))
    for t, fill in zip(bufs, (200, 3.0, 200, 3.0)):      # rows before and behind the chunk stay as they were
        assert (t[:, :11] == fill).all() and (t[:, 11 + n:] == fill).all()
    eng = _engine(B, H, G, D, n, "fp16")
    eng.prefill(x, y)
    a, b = torch.empty_like(x), torch.empty_like(x)
    eng.read_rows(a, None)
    _lib.check(lib.dc_q4_read_rows(bufs[0].data_ptr(), bufs[1].data_ptr(), rows, rows, P, D, 1, 11, None, 0, n, b.data_ptr(), st))
    assert torch.equal(a, b)
    moved = [torch.zeros(P, n, t.shape[2], dtype=t.dtype, device="cuda").copy_(t[:, 11:11 + n]) for t in bufs]
    ebits, sbits = torch.empty(B, H, n, dtype=torch.int32, device="cuda"), torch.empty(P, n, dtype=torch.int32, device="cuda")
    eng.score_rows(q, ebits)
    mm = torch.tensor([[-1, 0]] * P, dtype=torch.int32, device="cuda")
    _lib.check(lib.dc_q4_score_scan(moved[0].data_ptr(), moved[1].data_ptr(), n, P, n, D, 1, q.data_ptr(), 1, G, sbits.data_ptr(), n, mm.data_ptr(), st))
    assert torch.equal(ebits.reshape(P, n), sbits)
    assert torch.equal(mm, torch.stack([sbits.amin(1), sbits.amax(1)], 1))
    o1, o2 = torch.empty_like(q), torch.empty_like(q)
    eng.attend_rows(q, o1)
    scratch = torch.empty(int(lib.dc_q4_attend_scratch_bytes(P, G, D)), dtype=torch.uint8, device="cuda")
    _lib.check(lib.dc_q4_attend(*(t.data_ptr() for t in moved), n, n, P, H, G, D, 1, q.data_ptr(), None, 0, -1, 0, None, None, None, None,
                                None, 0, 0, 0, 0.0, o2.data_ptr(), None, None, None, scratch.data_ptr(), st))
    torch.cuda.synchronize()
    assert torch.equal(o1, o2)


@pytest.mark.parametrize("partials", [False, True])
def test_ragged_runs_never_read_what_nobody_wrote(partials):
    """Long unequal sequences through the stateless call with a scratch buffer full of NaN, as output and as partials."""
    from diffcache_b200 import _lib

    lib = _lib.load()
    B, H, G, D, n = 3, 2, 4, 128, 9000
    P = B * H
    x, y, q = _rows((B, H, n, D), "bf16", 180, False), _rows((B, H, n, D), "bf16", 181, False), _rows((B, H * G, D), "bf16", 182, False)
    lens = torch.tensor([9000, 0, 700], dtype=torch.int32, device="cuda")
    st = int(torch.cuda.current_stream().cuda_stream)
    bufs = [torch.zeros((P, n, d), dtype=t, device="cuda") for _ in range(2) for d, t in ((D // 2, torch.uint8), (D // 32, torch.bfloat16))]
    dx, dy, dq = x.cuda(), y.cuda(), q.cuda()
    _lib.check(lib.dc_q4_write_rows(dx.data_ptr(), dy.data_ptr(), H * n * D, n * D, D, P, H, n, D, 0, *(t.data_ptr() for t in bufs), n, 0, st))
    out = torch.full_like(dq, 7.0)
    acc, ml = torch.full((B, H * G, D), 7.0, device="cuda"), torch.full((B, H * G, 2), 7.0, device="cuda")
    scratch = torch.full((int(lib.dc_q4_attend_scratch_bytes(P, G, D)) // 4,), math.nan, device="cuda")
    dst = (None, None, acc.data_ptr(), ml.data_ptr()) if partials else (out.data_ptr(), None, None, None)
    _lib.check(lib.dc_q4_attend(*(t.data_ptr() for t in bufs), n, n, P, H, G, D, 0, dq.data_ptr(), None, 0, -1, 0, lens.data_ptr(),
                                None, None, None, None, 0, 0, 0, 0.0, *dst, scratch.data_ptr(), st))
    if partials:
        _lib.check(lib.dc_lse_combine(acc.data_ptr(), acc.numel(), ml.data_ptr(), ml.numel(), 1, B * H * G, D, 0, out.data_ptr(), None, st))
    torch.cuda.synchronize()
    for b in range(B):
        m = int(lens[b])
        for h in range(H):
            got = out[b, h * G:(h + 1) * G].cpu()[None]
            if m == 0:
                assert (got == 0).all()
                continue
            want, _, tol, _ = q4_util.attend(q[b, h * G:(h + 1) * G][None], q4_util.stored(x[b, h, :m])[None],
                                             q4_util.stored(y[b, h, :m])[None], torch.ones(1, m, dtype=torch.bool), D ** -0.5)
            q4_util.assert_close(got, want, tol, f"out {b},{h}")


@pytest.mark.parametrize("B,H,G,D,n", [(1, 2, 4, 128, 20001), (1, 1, 8, 256, 9000), (1, 3, 1, 64, 12345), (2, 1, 12, 128, 7000)])
def test_attend_many_partials(B, H, G, D, n):
    """Few problems with many rows: more CTAs than a cluster holds, merged by a second kernel."""
    _attend_case(B, H, G, D, n, "bf16", 190, res=130, new=True)
    _attend_case(B, H, G, D, n, "fp16", 191)
    _attend_case(B, H, G, D, n, "bf16", 192, lens=torch.tensor([n - 3, 100][:B], dtype=torch.int32), res=2)
    gen = torch.Generator().manual_seed(4)
    ids = torch.stack([torch.randperm(n, generator=gen)[:6500] for _ in range(B * H)]).reshape(B, H, 6500).to(torch.int32)
    _attend_case(B, H, G, D, n, "fp16", 193, ids=ids, new=True)


def test_adaptive_budget_on_a_4_bit_store():
    """The k-check works on the 4-bit scan's keys, and attention stops at its budget."""
    B, H, G, D, n, topk = 1, 3, 4, 128, 2000, 400
    x, y, q = _rows((B, H, n, D), "bf16", 200, False), _rows((B, H, n, D), "bf16", 201, False), _rows((B, H * G, D), "bf16", 202, False)
    q[:, :G] += x[0, 0, 5] * 0.5          # a head group whose mass sits on few rows
    eng = _engine(B, H, G, D, n, adaptive_budget=True, k_check_seq=[25, 50, 100, 200], attn_mass_threshold=0.5)
    eng.prefill(x.cuda(), y.cuda())
    out, idx = torch.empty_like(q, device="cuda"), torch.empty(B, H, topk, dtype=torch.int32, device="cuda")
    eng.decode_attend(q.cuda(), out, topk, out_idx=idx)
    budget = eng.last_budget()
    assert budget.min() >= 1 and budget.max() <= topk
    ks, vs = q4_util.stored(x), q4_util.stored(y)
    for h in range(H):
        pick = idx[0, h, :int(budget[0, h])].cpu().long()
        want, _, tol, _ = q4_util.attend(q[0, h * G:(h + 1) * G][None], ks[0, h][pick][None], vs[0, h][pick][None],
                                         torch.ones(1, len(pick), dtype=torch.bool), D ** -0.5)
        q4_util.assert_close(out[0, h * G:(h + 1) * G].cpu()[None], want, tol, f"head {h}")


def test_offsets_beyond_32_bits():
    """Rows more than 4 GB into a problem's codes: written, read back, scored and attended."""
    from diffcache_b200 import _lib

    lib = _lib.load()
    G, D, rows, n = 4, 128, 68_000_000, 300
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 12 GB of device memory")
    first = rows - n
    x, y, q = _rows((1, 1, n, D), "bf16", 210), _rows((1, 1, n, D), "bf16", 211), _rows((1, G, D), "bf16", 212, False)
    dx, dy, dq = x.cuda(), y.cuda(), q.cuda()
    st = int(torch.cuda.current_stream().cuda_stream)
    bufs = [torch.full((1, rows, d), fill, dtype=t, device="cuda") for _ in range(2)
            for d, t, fill in ((D // 2, torch.uint8, 0x88), (D // 32, torch.bfloat16, 0.0))]
    _lib.check(lib.dc_q4_write_rows(dx.data_ptr(), dy.data_ptr(), 0, 0, D, 1, 1, n, D, 0, *(t.data_ptr() for t in bufs), rows, first, st))
    back = torch.empty_like(dx)
    _lib.check(lib.dc_q4_read_rows(bufs[2].data_ptr(), bufs[3].data_ptr(), rows, rows, 1, D, 0, first, None, 0, n, back.data_ptr(), st))
    assert bit_rows(back, q4_util.stored(y).to(y.dtype))
    mean = dq.float().mean(1).to(dq.dtype).contiguous()
    bits = torch.zeros(rows, dtype=torch.int32, device="cuda")
    _lib.check(lib.dc_q4_score_scan(bufs[0].data_ptr(), bufs[1].data_ptr(), rows, 1, rows, D, 0, mean.data_ptr(), 0, 1, bits.data_ptr(), rows, None, st))
    dist, tol = q4_util.scan(q4_util.stored(x).reshape(1, n, D), mean.cpu())
    q4_util.assert_close(bits[first:].cpu().view(torch.float32)[None], dist, tol, "dist")
    assert (bits[:first].view(torch.float32) == 65536.0).all()
    ids = torch.arange(first, rows, dtype=torch.int32, device="cuda")
    out = torch.empty_like(dq)
    scratch = torch.empty(int(lib.dc_q4_attend_scratch_bytes(1, G, D)), dtype=torch.uint8, device="cuda")
    _lib.check(lib.dc_q4_attend(*(t.data_ptr() for t in bufs), rows, rows, 1, 1, G, D, 0, dq.data_ptr(), ids.data_ptr(), n, n, 0, None,
                                None, None, None, None, 0, 0, 0, 0.0, out.data_ptr(), None, None, None, scratch.data_ptr(), st))
    want, _, wtol, _ = q4_util.attend(q, q4_util.stored(x)[0], q4_util.stored(y)[0], torch.ones(1, n, dtype=torch.bool), D ** -0.5)
    q4_util.assert_close(out.cpu(), want, wtol, "ids")
    # every row: the zero rows in front score 0 and weigh in with values of 0
    _lib.check(lib.dc_q4_attend(*(t.data_ptr() for t in bufs), rows, rows, 1, 1, G, D, 0, dq.data_ptr(), None, 0, -1, 0, None,
                                None, None, None, None, 0, 0, 0, 0.0, out.data_ptr(), None, None, None, scratch.data_ptr(), st))
    x64 = torch.matmul(q[0].double(), q4_util.stored(x)[0, 0].T) * D ** -0.5
    e = torch.exp(x64)
    total = e.sum(-1, keepdim=True) + first
    ref = torch.matmul(e, q4_util.stored(y)[0, 0]) / total
    spread = torch.matmul(e, q4_util.stored(y)[0, 0].abs()) / total
    # a warp adds its share of the rows 16 at a time, each step off by at most 2^-23 of the running sum; at least 255 CTAs of
    # four warps share the rows
    rel = rows / (4 * 255 * 16) * 2.0 ** -23 + 2.0 ** -12
    q4_util.assert_close(out.cpu()[0], ref, rel * spread + 2.0 ** -8 * ref.abs() + 2.0 ** -30, "all")


def test_inputs_that_would_be_read_wrongly_are_refused():
    B, H, G, D, n = 2, 2, 2, 64, 10
    eng = _engine(B, H, G, D, 16)
    x = _rows((B, H, n, D), "bf16", 220)
    eng.prefill(x.cuda(), x.cuda())
    q = _rows((1, H * G, D), "bf16", 221, False).cuda()
    out = torch.empty(B, H * G, D, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="expanded"):
        eng.attend_rows(q.expand(B, H * G, D), out)
    kn = q[:, :H].contiguous()
    with pytest.raises(ValueError, match="expanded"):
        eng.attend_rows(q.repeat(B, 1, 1), out, k_new=kn.expand(B, H, D), v_new=kn.expand(B, H, D))
    for shape in ((B, H, 1, D),):          # a host row whose row stride means nothing
        row = torch.zeros(shape, dtype=torch.bfloat16)
        eng.write_rows(n, row, row)
    assert eng.ctx_len == n + 1
    from diffcache_b200 import DiffCacheGPU

    wide = DiffCacheGPU(B, H * G, H, D, max_ctx_len=16)
    wide.write_rows(0, row, row)
    wide.write_rows(1, util.u16(x), util.u16(x))
    back = torch.empty(B, H, n, D, dtype=torch.bfloat16, device="cuda")
    wide.read_rows(back, None, row0=1)
    assert torch.equal(back.cpu(), x)


def test_refusals():
    from diffcache_b200 import DiffCacheError

    B, H, G, D, n = 1, 2, 4, 128, 20
    eng = _engine(B, H, G, D, 32)
    x = _rows((B, H, n, D), "bf16", 170).cuda()
    eng.prefill(x, x)
    q, out = _rows((B, H * G, D), "bf16", 171, False).cuda(), torch.empty(B, H * G, D, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(TypeError, match="expected torch.bfloat16"):
        eng.write_rows(0, x.to(torch.float16), x.to(torch.float16))
    with pytest.raises(DiffCacheError, match="gap"):
        eng.write_rows(21, x[:, :, :1], x[:, :, :1])
    with pytest.raises(DiffCacheError, match="exceed"):
        eng.write_rows(13, x, x)
    with pytest.raises(DiffCacheError, match="aligned|multiples"):
        t = torch.zeros(B, H, n, D + 4, dtype=torch.bfloat16, device="cuda")[..., :D]
        eng.write_rows(0, t, t)
    with pytest.raises(ValueError, match="head_dim axis"):
        t = torch.zeros(B, H, n, 2 * D, dtype=torch.bfloat16, device="cuda")[..., ::2]
        eng.write_rows(0, t, t)
    with pytest.raises(ValueError, match="shape"):
        eng.write_rows(0, x[..., :64], x[..., :64])
    with pytest.raises(ValueError, match="contiguous"):
        eng.read_rows(torch.empty(B, H, D, n, dtype=torch.bfloat16, device="cuda").transpose(2, 3), None)
    with pytest.raises(ValueError, match="device tensor"):
        eng.read_rows(torch.empty(B, H, n, D, dtype=torch.bfloat16), None)
    with pytest.raises(DiffCacheError, match="exceed"):
        eng.read_rows(x.clone(), None, row0=20)
    with pytest.raises(TypeError, match="expected one of"):
        eng.read_rows(x.clone(), None, ids=torch.zeros(B, H, n, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="shape"):
        eng.score_rows(q[:, :3], torch.empty(B, H, n, dtype=torch.int32, device="cuda"))
    with pytest.raises(DiffCacheError, match="max_ctx_len"):
        eng.score_rows(q, torch.empty(B, H, 33, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="ids or lens"):
        eng.attend_rows(q, out, ids=torch.zeros(B, H, 1, dtype=torch.int32, device="cuda"), lens=torch.zeros(B, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="pairs"):
        eng.attend_rows(q, out, k_new=q[:, :H].contiguous())
    with pytest.raises(ValueError, match="hold"):
        eng.attend_rows(q, out, res_k=x, res_v=x, res_len=n, k_new=q[:, :H].contiguous(), v_new=q[:, :H].contiguous())
    with pytest.raises(ValueError, match="res_len > 0"):
        eng.attend_rows(q, out, res_len=1)
    with pytest.raises(TypeError, match="expected"):
        eng.attend_rows(q, out, out_lse=torch.empty(B, H * G, dtype=torch.float16, device="cuda"))
    with pytest.raises(DiffCacheError, match="4 bits"):
        from diffcache_b200 import _lib
        buf = np.empty((B, H, n, D), np.uint16)
        _lib.check(eng._lib.dc_export_rows(eng._h, buf.ctypes.data, buf.ctypes.data))
