"""Rotary positions, the paged cache's append / gather and attention over it,
against 64-bit references (paged_cases.py)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import paged_cases as P

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
U = 2.0 ** -8  # bf16 rounds within U of a value


def table(lmx, kind, positions, rot, theta=1e4, factor=8.0, low=1.0, high=4.0, orig=512.0, attn=0.0):
    c = torch.empty(positions, rot // 2, device="cuda")
    s = torch.empty_like(c)
    sc = lmx.RopeScaling(kind, theta, factor, low, high, orig, attn)
    lmx.call("lmx_rope_table", sc, positions, rot, c.data_ptr(), s.data_ptr(), None)
    return c, s


def desc(lmx, c, s, inter):
    return lmx.RopeDesc(c.data_ptr(), s.data_ptr(), c.shape[0], 2 * c.shape[1], inter)


def turn(x, c, s, inter):
    """64-bit rotation of x [tokens, heads, dim] by rows c, s [tokens, rot / 2]."""
    x, c, s = x.double(), c.double()[:, None], s.double()[:, None]
    r, y = 2 * c.shape[-1], x.clone()
    ia = torch.arange(0, r, 2) if inter else torch.arange(r // 2)
    ib = ia + (1 if inter else r // 2)
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y


# ---------------------------------------------------------------- rotation
@pytest.mark.parametrize("kind", range(4))
@pytest.mark.parametrize("rot", [16, 64, 128])
def test_rope_table(lmx, cuda, kind, rot):
    # yarn's bounds are turns: 32 and 1
    low, high = (1.0, 32.0) if kind == 3 else (1.0, 4.0)
    n = 1031
    c, s = table(lmx, kind, n, rot, low=low, high=high)
    f = 1e4 ** (-np.arange(0, rot, 2) / rot)
    mul = 1.0
    if kind == 1:
        f = f / 8
    elif kind == 2:
        for i, v in enumerate(f):
            wl = 2 * math.pi / v
            if wl > 512 / low:
                f[i] = v / 8
            elif wl > 512 / high:
                k = (512 / wl - low) / (high - low)
                f[i] = (1 - k) * v / 8 + k * v
    elif kind == 3:
        a, b = (rot * math.log(512 / (t * 2 * math.pi)) / (2 * math.log(1e4)) for t in (32.0, 1.0))
        a, b = max(math.floor(a), 0), min(math.ceil(b), rot - 1)
        k = np.clip((np.arange(rot // 2) - a) / max(b - a, 1e-3), 0, 1)
        f = f / 8 * k + f * (1 - k)
        mul = 0.1 * math.log(8.0) + 1
    ang = np.arange(n)[:, None] * f
    # one rounding to fp32 (at most 2^-24 times a value below 2), plus the angle's 64-bit error
    for got, want in ((c, np.cos(ang) * mul), (s, np.sin(ang) * mul)):
        assert np.abs(got.cpu().double().numpy() - want).max() <= 2.0 ** -24 * max(mul, 1.0) + 1e-11


# tokens, heads, dim, rot, in place, extra row width
@pytest.mark.parametrize("n,h,d,rot,place,extra", [
    (1, 1, 64, 64, 0, 0), (1, 5, 128, 64, 1, 8), (7, 3, 128, 128, 0, 384), (33, 9, 128, 96, 1, 0),
    (130, 4, 64, 16, 0, 64), (5, 2, 256, 128, 1, 16), (3, 4, 80, 32, 0, 0)])
@pytest.mark.parametrize("inter", [0, 1])
@pytest.mark.parametrize("inverse", [0, 1])
def test_rope_apply(lmx, cuda, n, h, d, rot, place, extra, inter, inverse):
    gen = torch.Generator().manual_seed(n * 7 + rot)
    c, s = table(lmx, 0, 200, rot)
    x = torch.randn((n, h * d + extra), generator=gen).to(BF16)
    pos = torch.randint(0, 200, (n,), generator=gen, dtype=torch.int32)
    pos[0] = 199 if n > 1 else 0
    dx, dp = x.cuda(), pos.cuda()
    y = dx if place else torch.full((n, h * d), 7.0, dtype=BF16, device="cuda")
    lmx.call("lmx_rope_apply", desc(lmx, c, s, inter), dx.data_ptr(), x.stride(0), dp.data_ptr(), n, h, d, inverse,
             y.data_ptr(), y.stride(0), None)
    got = y.cpu()[:, :h * d].reshape(n, h, d)
    rows = x[:, :h * d].reshape(n, h, d)
    cc, ss = c.cpu()[pos.long()], s.cpu()[pos.long()]
    want = turn(rows, cc, -ss if inverse else ss, inter)
    # two products and a sum in fp32, each within 2^-24 of terms at most |a| + |b|, then one bf16 rounding
    amax = rows.double().abs().amax(-1, keepdim=True) * 2
    assert ((got.double() - want).abs() <= U * want.abs() + 2.0 ** -22 * amax).all()
    assert torch.equal(got[..., rot:], rows[..., rot:])
    if place and extra:
        assert torch.equal(y.cpu()[:, h * d:], x[:, h * d:])


@pytest.mark.parametrize("inter", [0, 1])
def test_rope_gradient(lmx, cuda, inter):
    # the rotation is linear: its matrix by differences (unit steps from zero)
    # against the matrix of its gradient, entry for entry
    d, rot = 64, 48
    c, s = table(lmx, 2, 64, rot)
    e = torch.eye(d, dtype=BF16, device="cuda")
    pos = torch.full((d,), 37, dtype=torch.int32, device="cuda")
    out = []
    for inverse in (0, 1):
        y = torch.empty_like(e)
        lmx.call("lmx_rope_apply", desc(lmx, c, s, inter), e.data_ptr(), d, pos.data_ptr(), d, 1, d, inverse,
                 y.data_ptr(), d, None)
        out.append(y.cpu())
    assert torch.equal(out[0].T, out[1])
    gen = torch.Generator().manual_seed(1)
    g = torch.randn((d, 1, d), generator=gen).to(BF16)
    y = torch.empty_like(e)
    dg = g.cuda()
    lmx.call("lmx_rope_apply", desc(lmx, c, s, inter), dg.data_ptr(), d, pos.data_ptr(), d, 1, d, 1, y.data_ptr(), d, None)
    want = g.double()[:, 0] @ turn(torch.eye(d)[:, None], c.cpu()[37:38].expand(d, -1), s.cpu()[37:38].expand(d, -1), inter)[:, 0].T
    amax = g.double().abs().amax(-1) * 2
    assert ((y.cpu().double() - want).abs() <= U * want.abs() + 2.0 ** -22 * amax).all()


def test_rope_position_outside(lmx, cuda):
    c, s = table(lmx, 0, 16, 64)
    x = torch.randn(3, 2, 64, device="cuda").to(BF16)
    y = torch.full_like(x, 5.0)
    pos = torch.tensor([3, 16, -1], dtype=torch.int32, device="cuda")
    P.device_error(lmx)
    lmx.call("lmx_rope_apply", desc(lmx, c, s, 0), x.data_ptr(), 128, pos.data_ptr(), 3, 2, 64, 0, y.data_ptr(), 128, None)
    cuda.cuda.synchronize()
    assert P.device_error(lmx) == 0x44
    assert (y[1:] == 5.0).all() and not (y[0] == 5.0).all()


# ------------------------------------------------------------------ append
LENS = {"one": [(1, 1)], "first": [(5, 5)], "ragged": [(1, 70), (0, 40), (37, 37), (3, 131), (0, 0), (16, 64)],
        "empty rows": [(4, 2), (3, 0), (2, 66)]}


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("lens,hk,g,d,page,rot,inter,norm,gap,pad", [
    ("one", 1, 1, 128, 16, 128, 0, 0, 0, 0), ("first", 2, 3, 64, 32, 64, 1, 1, 0, 3),
    ("ragged", 2, 4, 128, 16, 128, 0, 1, 16, 0), ("ragged", 3, 1, 64, 64, 32, 0, 0, 0, 1),
    ("ragged", 1, 5, 128, 128, 64, 1, 0, 32, 2), ("empty rows", 2, 2, 128, 32, 96, 0, 0, 0, 0),
    ("ragged", 8, 4, 128, 256, 0, 0, 0, 0, 0)])
def test_append_and_gather(lmx, cuda, bits, lens, hk, g, d, page, rot, inter, norm, gap, pad):
    cache = P.Cache(3, LENS[lens], hk, d, bits, page, gap=gap, pad=pad)
    kv, batch = cache.device(lmx, zero_stride=gap == 0)
    n, heads = cache.tokens, hk * g
    x = torch.randn((n, (heads + 2 * hk) * d + 8), generator=cache.gen).to(BF16)
    dx = x.cuda()
    wn = [(1 + 0.3 * torch.randn(d, generator=cache.gen)).to(BF16) for _ in "qk"]
    dw = [w.cuda() for w in wn]
    if rot:
        c, s = table(lmx, 0, 256, rot)
    qo = torch.full((n, heads * d + 16), 9.0, dtype=BF16, device="cuda")
    P.device_error(lmx)
    lmx.call("lmx_paged_append", kv, batch, desc(lmx, c, s, inter) if rot else None, dx.data_ptr(),
             dx.data_ptr() + 2 * heads * d, dx.data_ptr() + 2 * (heads + hk) * d, x.stride(0), heads,
             dw[0].data_ptr() if norm else None, dw[1].data_ptr() if norm else None, 1e-5, qo.data_ptr(), qo.stride(0), None)
    ko, vo = (torch.full((n, hk, d), 9.0, dtype=BF16, device="cuda") for _ in "kv")
    lmx.call("lmx_paged_gather", kv, batch, ko.data_ptr(), vo.data_ptr(), None)
    cuda.cuda.synchronize()
    assert P.device_error(lmx) == 0
    q, k, v = (t.reshape(n, -1, d) for t in (x[:, :heads * d], x[:, heads * d:(heads + hk) * d],
                                             x[:, (heads + hk) * d:(heads + 2 * hk) * d]))
    touched = {m: torch.zeros(len(cache.pool[m]), dtype=torch.bool) for m in "kv"}
    after = {m: t.cpu() for m, t in cache.dev.items()}
    got_q = qo.cpu()[:, :heads * d].reshape(n, heads, d)
    assert (qo.cpu()[:, heads * d:] == 9.0).all()
    for i, (new, rows) in enumerate(cache.lens):
        for t in range(new):
            at, pos = cache.start[i] + t, rows - new + t
            if pos < 0:
                assert (got_q[at] == 0).all() and (ko[at] == 0).all() and (vo[at] == 0).all()
                continue
            want = []
            for y, w in ((q[at], wn[0]), (k[at], wn[1])):
                y = y.double()
                if norm:
                    y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
                if rot:
                    y = turn(y[None], c.cpu()[pos:pos + 1], s.cpu()[pos:pos + 1], inter)[0]
                want.append(y)
            # fp32 arithmetic: the norm's sum of d squares (d 2^-24), five more roundings, the rotation's three
            amax = max(w.abs().max().item() for w in want) * 2
            slack = (d + 8) * 2.0 ** -24 * amax
            assert ((got_q[at].double() - want[0]).abs() <= U * want[0].abs() + slack).all()
            r = cache.at(i, torch.tensor([pos]))[0]
            for m, y, back in (("k", want[1], ko), ("v", v[at].double(), vo)):
                touched[m][r] = True
                if bits == 16:
                    assert ((after[m][r].double() - y).abs() <= U * y.abs() + (slack if m == "k" else 0)).all()
                    assert torch.equal(back[at].cpu(), after[m][r])
                    continue
                sc, bi = after[m + "s"][r], after[m + "b"][r]
                val = P.values(after[m][r], sc, bi, bits)
                # half a step, the bias's rounding (values below it clamp to code 0, and the
                # codes end that much below the maximum), the scale's rounding over all steps
                grp = y.unflatten(-1, (-1, 64))
                lo, span = grp.amin(-1), grp.amax(-1) - grp.amin(-1)
                lim = 0.5 * sc.double() + U * lo.abs() + U * span + 2 * slack
                assert ((val - y).abs().unflatten(-1, (-1, 64)) <= lim[..., None]).all()
                top = (1 << bits) - 1
                assert ((sc.double() - span / top).abs() <= U * span / top + slack).all()
                assert ((bi.double() - lo).abs() <= U * lo.abs() + slack).all()
                assert torch.equal(back[at].cpu(), val.float().to(BF16))
                if m == "v":  # unrotated rows quantize exactly by the cache's rule
                    cq, cs, cb = P.quantize(v[at].float(), bits)
                    assert torch.equal(after[m][r], P.pack(cq, bits)) and torch.equal(sc, cs) and torch.equal(bi, cb)
    for m, t in after.items():  # every other row as it was
        keep = ~touched[m[0]]
        assert torch.equal(t[keep].view(torch.int16 if t.dtype == BF16 else torch.uint8),
                           cache.pool[m][keep].view(torch.int16 if t.dtype == BF16 else torch.uint8))
    assert (got_q[cache.start[-1]:] == 9.0).all() and (ko[cache.start[-1]:] == 9.0).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("inter", [0, 1])
@pytest.mark.parametrize("rot", [64, 128])
def test_rotated_codes_are_those_of_fp32(lmx, cuda, bits, inter, rot):
    # every product, sum and quotient of the rule rounded by itself in fp32: the codes come out the same
    cache = P.Cache(4, [(500, 700)], 4, 128, bits, 32)
    kv, batch = cache.device(lmx)
    c, s = table(lmx, 0, 1024, rot)
    x = torch.randn((500, 8 * 128), generator=cache.gen).to(BF16)
    dx = x.cuda()
    lmx.call("lmx_paged_append", kv, batch, desc(lmx, c, s, inter), None, dx.data_ptr(), dx.data_ptr() + 1024, 1024, 0, None,
             None, 0.0, None, 0, None)
    cc, ss = c.cpu()[200:700, None], s.cpu()[200:700, None]
    k = x[:, :512].reshape(500, 4, 128).float()
    ia = torch.arange(0, rot, 2) if inter else torch.arange(rot // 2)
    ib = ia + (1 if inter else rot // 2)
    y = k.clone()
    y[..., ia] = k[..., ia] * cc - k[..., ib] * ss
    y[..., ib] = k[..., ib] * cc + k[..., ia] * ss
    at = cache.at(0, torch.arange(200, 700))
    for m, v in (("k", y), ("v", x[:, 512:].reshape(500, 4, 128).float())):
        q, sc, bi = P.quantize(v, bits)
        assert torch.equal(cache.dev[m].cpu()[at], P.pack(q, bits))
        assert torch.equal(cache.dev[m + "s"].cpu()[at], sc) and torch.equal(cache.dev[m + "b"].cpu()[at], bi)


def test_append_in_place_and_without_queries(lmx, cuda):
    cache = P.Cache(5, [(3, 9), (2, 2)], 2, 128, 16, 16)
    kv, batch = cache.device(lmx)
    c, s = table(lmx, 0, 32, 128)
    x = torch.randn((5, 8 * 128), generator=cache.gen).to(BF16)
    a, b = x.cuda(), x.cuda()
    r = desc(lmx, c, s, 0)
    out = torch.empty((5, 512), dtype=BF16, device="cuda")
    lmx.call("lmx_paged_append", kv, batch, r, a.data_ptr(), a.data_ptr() + 1024, a.data_ptr() + 1536, 1024, 4, None,
             None, 0.0, out.data_ptr(), 512, None)
    first = cache.dev["k"].clone()
    lmx.call("lmx_paged_append", kv, batch, r, b.data_ptr(), b.data_ptr() + 1024, b.data_ptr() + 1536, 1024, 4, None,
             None, 0.0, b.data_ptr(), 1024, None)
    assert torch.equal(b[:, :512], out) and torch.equal(b[:, 512:].cpu(), x[:, 512:])
    cache.dev["k"].fill_(0)
    lmx.call("lmx_paged_append", kv, batch, r, None, a.data_ptr() + 1024, a.data_ptr() + 1536, 1024, 0, None, None, 0.0,
             None, 0, None)
    at = torch.cat([cache.at(0, torch.arange(6, 9)), cache.at(1, torch.arange(2))])
    assert torch.equal(cache.dev["k"].cpu()[at], first.cpu()[at])


@pytest.mark.parametrize("fault", ["page", "table", "positions"])
def test_append_without_a_row(lmx, cuda, fault):
    cache = P.Cache(6, [(2, 40), (2, 20)], 1, 64, 16, 16, spare=0)
    if fault == "page":
        cache.table[0, 2] = cache.pages  # rows 32..47 of sequence 0
    kv, batch = cache.device(lmx)
    if fault == "table":
        cache.index[1][0] = 16 * cache.table.shape[1] + 2  # two tokens past the table
    c, s = table(lmx, 0, 38 if fault == "positions" else 64, 64)
    x = torch.ones((4, 3 * 64), dtype=BF16, device="cuda")
    qo = torch.full((4, 64), 9.0, dtype=BF16, device="cuda")
    P.device_error(lmx)
    lmx.call("lmx_paged_append", kv, batch, desc(lmx, c, s, 0), x.data_ptr(), x.data_ptr() + 128, x.data_ptr() + 256, 192,
             1, None, None, 0.0, qo.data_ptr(), 64, None)
    cuda.cuda.synchronize()
    assert P.device_error(lmx) == 0x44
    assert (qo[:2] == 0).all() and not (qo[2:] == 0).all()
    good = cache.at(1, torch.arange(18, 20)).flatten()
    keep = torch.ones(len(cache.pool["k"]), dtype=torch.bool)
    keep[good] = False
    now = cache.dev["v"].cpu()
    assert (now[good] == 1).all() and torch.equal(now[keep].view(torch.int16), cache.pool["v"][keep].view(torch.int16))


# --------------------------------------------------------------- attention
def attend(lmx, cache, q, heads, scale, window, with_lse=True, extra=0, stream=None):
    kv, batch = cache.device(lmx)
    n, d = cache.tokens, cache.dim
    dq = torch.zeros((n, heads * d + extra), dtype=BF16)
    dq[:, :heads * d] = q.reshape(n, -1)
    dq = dq.cuda()
    out = torch.full((n, heads * d + 2 * extra), 9.0, dtype=BF16, device="cuda")
    lse = torch.full((n, heads), 9.0, device="cuda")
    size = lmx.lib().lmx_paged_attention_scratch_bytes(kv, batch, heads)
    scratch = torch.randint(0, 255, (size,), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    lmx.call("lmx_paged_attention", kv, batch, dq.data_ptr(), dq.stride(0), heads, scale, window, scratch.data_ptr(), size,
             out.data_ptr(), out.stride(0), lse.data_ptr() if with_lse else None, stream)
    torch.cuda.synchronize()
    assert (out[:, heads * d:] == 9.0).all()
    return out[:, :heads * d].reshape(n, heads, d).cpu(), lse.cpu()


def code_span(cache):
    """Per sequence and KV head, the largest |scale| * 280 + |bias| of K: what the codes' products are sums of."""
    if cache.bits == 16:
        return None
    return [(280 * cache.pool["ks"][cache.at(i, torch.arange(m))].double().abs()
             + cache.pool["kb"][cache.at(i, torch.arange(m))].double().abs()).max().item() if m > 0 else 0.0
            for i, (_, m) in enumerate(cache.lens)]


def check(cache, q, got, lse, scale, window, p_err=2.0 ** -16, kv_err=0.0):
    """Bounds: fp32 products and sums of dim terms put a score off by at most dim 2^-24 of the sum of their sizes (Q; for
    quantized K the codes' sums stand in its place), so p by twice that (numerator and denominator), p_err more where
    p enters P V rounded, kv_err where K and V do; 2^-20 for the exponentials and sums; then one bf16 rounding."""
    want, wl, A, Q = P.attention(cache, q, scale, window)
    span = code_span(cache)
    if span is not None:
        for i in range(len(cache.lens)):
            at = slice(cache.start[i], cache.start[i + 1])
            Q[at] = q[at].double().abs().sum(-1) * span[i] * scale
    n = cache.start[-1]
    ds = Q[:n] * (cache.dim * 2.0 ** -24) + P.attention(cache, q, scale, window)[3][:n] * kv_err
    err = (got[:n].double() - want[:n]).abs()
    lim = U * want[:n].abs() + A[:n] * (p_err + kv_err + 2 * ds + 2.0 ** -20)[..., None] * (1 + U)
    assert (err <= lim).all(), (err / lim.clamp(min=1e-30)).max()
    fin = wl[:n] > -math.inf
    assert torch.equal(fin, lse[:n] > -math.inf) and not torch.isnan(lse[:n]).any()
    dl = (lse[:n].double() - wl[:n])[fin].abs()
    assert (dl <= (ds[fin] + 2.0 ** -20 * (1 + wl[:n][fin].abs()))).all(), dl.max()
    assert (got[:n][~fin] == 0).all()


FEW = {"one": [(1, 1)], "two": [(2, 2)], "edge": [(1, 16), (1, 17), (1, 64), (1, 65), (1, 15)],
       "ragged": [(1, 300), (0, 40), (3, 131), (2, 2), (0, 0), (4, 64), (1, 1)],
       "empty rows": [(4, 2), (3, 0), (2, 66), (1, 0)], "long": [(1, 2500)], "split": [(2, 1500), (1, 5)]}


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("lens,hk,g,d,page,window", [
    ("one", 1, 1, 128, 16, 0), ("two", 2, 3, 64, 32, 0), ("edge", 2, 4, 128, 16, 0), ("edge", 2, 7, 64, 64, 20),
    ("ragged", 2, 4, 128, 32, 0), ("ragged", 1, 3, 64, 128, 33), ("ragged", 3, 2, 128, 256, 1),
    ("empty rows", 2, 2, 128, 32, 0), ("empty rows", 1, 4, 64, 16, 5), ("long", 1, 16, 128, 16, 0),
    ("long", 2, 1, 64, 128, 700), ("split", 1, 5, 128, 64, 0), ("split", 4, 8, 128, 16, 129)])
def test_attention_few_rows(lmx, cuda, bits, lens, hk, g, d, page, window):
    cache = P.Cache(11, FEW[lens], hk, d, bits, page, gap=16 if g == 3 else 0, pad=2 if g == 7 else 0)
    q = (torch.randn((cache.tokens, hk * g, d), generator=cache.gen) * 1.5).to(BF16)
    P.device_error(lmx)
    got, lse = attend(lmx, cache, q, hk * g, d ** -0.5, window, extra=8 if g == 2 else 0)
    assert P.device_error(lmx) == 0
    check(cache, q, got, lse, d ** -0.5, window)


@pytest.fixture
def prompt_rows(lmx):
    """Set the row count from which the prompt kernel runs; restores the default."""
    before = lmx.lib().lmx_paged_prompt_min_rows()
    yield lambda n: lmx.call("lmx_set_paged_prompt_min_rows", n)
    lmx.call("lmx_set_paged_prompt_min_rows", before)


PROMPT = {"one": [(1, 1)], "prompt": [(200, 200)], "tile edges": [(128, 128), (129, 129), (127, 256), (64, 64), (32, 383)],
          "ragged": [(150, 300), (0, 40), (1, 131), (2, 2), (0, 0), (77, 640), (1, 1), (300, 301)],
          "empty rows": [(40, 20), (30, 0), (2, 66), (1, 0), (200, 10)], "long": [(40, 3000)],
          "mixed": [(1, 700), (90, 1200), (1, 17), (1, 128), (5, 129)]}


# rows at the 128-key tile's and the page's ends, every grouping (rows of a
# tile that 128 / G does not fill), windows that end inside a tile and a page
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("lens,hk,g,d,page,window", [
    ("one", 1, 1, 128, 16, 0), ("prompt", 2, 1, 64, 32, 0), ("prompt", 1, 4, 128, 128, 0), ("tile edges", 2, 4, 128, 16, 0),
    ("tile edges", 1, 3, 64, 64, 50), ("tile edges", 1, 1, 128, 256, 128), ("ragged", 2, 4, 128, 32, 0),
    ("ragged", 1, 7, 64, 128, 33), ("ragged", 3, 2, 128, 256, 1), ("ragged", 2, 5, 128, 64, 200),
    ("empty rows", 2, 2, 128, 32, 0), ("empty rows", 1, 4, 64, 16, 5), ("long", 1, 8, 128, 16, 0),
    ("long", 2, 16, 64, 128, 700), ("mixed", 2, 8, 128, 16, 0), ("mixed", 1, 64, 64, 64, 129), ("mixed", 4, 1, 64, 16, 0)])
def test_attention_prompt_kernel(lmx, cuda, prompt_rows, bits, lens, hk, g, d, page, window):
    prompt_rows(1)
    cache = P.Cache(21, PROMPT[lens], hk, d, bits, page, gap=16 if g == 3 else 0, pad=2 if g == 7 else 0)
    q = (torch.randn((cache.tokens, hk * g, d), generator=cache.gen) * 1.5).to(BF16)
    P.device_error(lmx)
    got, lse = attend(lmx, cache, q, hk * g, d ** -0.5, window, extra=8 if g == 2 else 0)
    assert P.device_error(lmx) == 0
    # p enters P V as bf16: 2^-8; over a quantized cache p and the K and V values are fp16: 2^-11
    if bits == 16:
        check(cache, q, got, lse, d ** -0.5, window, p_err=2.0 ** -8)
    else:
        check(cache, q, got, lse, d ** -0.5, window, p_err=2.0 ** -11, kv_err=2.0 ** -11)


def test_attention_prompt_kernel_large_scores(lmx, cuda, prompt_rows):
    prompt_rows(1)
    cache = P.Cache(22, [(130, 333), (2, 64)], 2, 128, 16, 32, k_std=8.0)
    q = (torch.randn((132, 8, 128), generator=cache.gen) * 8).to(BF16)
    got, lse = attend(lmx, cache, q, 8, 0.25, 0)
    check(cache, q, got, lse, 0.25, 0, p_err=2.0 ** -8)


@pytest.mark.parametrize("rows", [1, 0])
def test_attention_nan_stays_in_its_rows(lmx, cuda, prompt_rows, rows):
    # a NaN query makes its own rows NaN and no others; a NaN key, every row that sees it
    prompt_rows(rows)
    cache = P.Cache(23, [(2, 300), (140, 140)], 1, 128, 16, 32)
    cache.pool["k"][cache.at(0, torch.tensor([117]))] = math.nan
    q = torch.randn((142, 2, 128), generator=cache.gen).to(BF16)
    q[10, 1, 5] = math.nan
    got, lse = attend(lmx, cache, q, 2, 0.1, 0)
    bad = torch.zeros(142, 2, dtype=torch.bool)
    bad[:2], bad[10, 1] = True, True
    assert torch.equal(torch.isnan(got).all(-1), bad) and torch.equal(torch.isnan(got).any(-1), bad)
    assert torch.equal(torch.isnan(lse), bad)


def test_attention_peaked_and_large_scores(lmx, cuda):
    # one key takes all the weight, and scores far apart (hundreds in the exponent)
    cache = P.Cache(12, [(1, 333), (2, 64)], 2, 128, 16, 32, k_std=8.0)
    q = (torch.randn((3, 8, 128), generator=cache.gen) * 8).to(BF16)
    got, lse = attend(lmx, cache, q, 8, 0.25, 0)
    check(cache, q, got, lse, 0.25, 0)


def test_attention_same_result_twice_and_on_a_stream(lmx, cuda):
    cache = P.Cache(13, [(1, 900), (3, 77), (1, 64)], 2, 128, 8, 64)
    q = torch.randn((5, 8, 128), generator=cache.gen).to(BF16)
    a, la = attend(lmx, cache, q, 8, 0.1, 0)
    st = torch.cuda.Stream()
    b, lb = attend(lmx, cache, q, 8, 0.1, 0, stream=st.cuda_stream)
    assert torch.equal(a, b) and torch.equal(la, lb)
    c, lc = attend(lmx, cache, q, 8, 0.1, 0, with_lse=False)
    assert torch.equal(a, c) and (lc == 9.0).all()


def test_attention_many_sequences(lmx, cuda):
    lens = [(i % 3, 1 + (i * 37) % 90) for i in range(300)]
    lens = [(min(n, r), r) for n, r in lens]
    cache = P.Cache(14, lens, 1, 64, 16, 16)
    q = torch.randn((cache.tokens, 2, 64), generator=cache.gen).to(BF16)
    got, lse = attend(lmx, cache, q, 2, 0.125, 0)
    check(cache, q, got, lse, 0.125, 0)


@pytest.mark.parametrize("rows", [0, 1])
def test_pages_past_four_gigabytes(lmx, cuda, prompt_rows, rows):
    # K and V interleaved in one pool of 4.7 GB (page_stride), the sequence's pages at its far end
    prompt_rows(rows)
    P_, hk, d, pages = 256, 1, 128, 36000
    pool = torch.zeros(pages * 2 * P_ * d, dtype=BF16, device="cuda")
    kv = lmx.PagedKvDesc(pages, P_, hk, d, 16, 2 * P_, pool.data_ptr(), pool.data_ptr() + P_ * d * 2)
    n = 300
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    batch = lmx.PagedBatch(1, n, n, start.data_ptr(), length.data_ptr(), table.data_ptr(), 2)
    gen = torch.Generator().manual_seed(2)
    x = torch.randn((n, 4, d), generator=gen).to(BF16).cuda()  # two q heads, k, v
    q = torch.empty((n, 2, d), dtype=BF16, device="cuda")
    lmx.call("lmx_paged_append", kv, batch, None, x.data_ptr(), x.data_ptr() + 4 * d, x.data_ptr() + 6 * d, 4 * d, 2, None,
             None, 0.0, q.data_ptr(), 2 * d, None)
    back = [torch.empty((n, 1, d), dtype=BF16, device="cuda") for _ in "kv"]
    lmx.call("lmx_paged_gather", kv, batch, back[0].data_ptr(), back[1].data_ptr(), None)
    assert torch.equal(q, x[:, :2]) and torch.equal(back[0], x[:, 2:3]) and torch.equal(back[1], x[:, 3:])
    at = (pages - 1) * 2 * P_ * d
    assert torch.equal(pool[at:at + P_ * d].view(P_, d), x[:P_, 2]) and torch.equal(pool[at + P_ * d:].view(P_, d), x[:P_, 3])
    size = lmx.lib().lmx_paged_attention_scratch_bytes(kv, batch, 2)
    scratch, out = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty_like(q)
    lmx.call("lmx_paged_attention", kv, batch, q.data_ptr(), 2 * d, 2, 0.09, 0, scratch.data_ptr(), size, out.data_ptr(),
             2 * d, None, None)
    z = torch.einsum("qhd,kd->hqk", x[:, :2].double(), x[:, 2].double()) * 0.09
    z.masked_fill_(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    p = torch.softmax(z, -1)
    want = torch.einsum("hqk,kd->qhd", p, x[:, 3].double())
    A = torch.einsum("hqk,kd->qhd", p, x[:, 3].double().abs())
    # bf16 output; p as bf16 in the prompt kernel; scores to 128 2^-24 of their terms' sum (below 2^5 here)
    assert ((out.double() - want).abs() <= U * want.abs() + A * (2.0 ** -8 + 2.0 ** -11)).all()


def test_calls_in_a_cuda_graph(lmx, cuda):
    cache = P.Cache(17, [(1, 200), (70, 300), (1, 33)], 2, 128, 8, 32)
    kv, batch = cache.device(lmx)
    n = cache.tokens
    c, s = table(lmx, 0, 512, 128)
    x = torch.randn((n, 12 * 128), generator=cache.gen).to(BF16).cuda()
    q, out = (torch.empty((n, 8 * 128), dtype=BF16, device="cuda") for _ in "qo")
    size = lmx.lib().lmx_paged_attention_scratch_bytes(kv, batch, 8)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")

    def step(stream):
        lmx.call("lmx_paged_append", kv, batch, desc(lmx, c, s, 0), x.data_ptr(), x.data_ptr() + 2048, x.data_ptr() + 2560,
                 12 * 128, 8, None, None, 0.0, q.data_ptr(), 1024, stream)
        lmx.call("lmx_paged_attention", kv, batch, q.data_ptr(), 1024, 8, 0.088, 0, scratch.data_ptr(), size, out.data_ptr(),
                 1024, None, stream)

    step(None)
    torch.cuda.synchronize()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    # the lengths are read on the device: the same graph serves other ones
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    cache.index[1][2] = 20
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[:71], first[:71]) and not torch.equal(out[71], first[71])


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("rows", [0, 1])
def test_pages_before_the_window_may_be_gone(lmx, cuda, prompt_rows, bits, rows):
    # rows that no query sees any more: their table entries name nothing, or a page of NaN
    prompt_rows(rows)
    lens, window = [(3, 300), (70, 500), (1, 20)], 50
    cache = P.Cache(18, lens, 2, 128, bits, 16, spare=0)
    for i, (new, n) in enumerate(lens):
        gone = max(0, n - new - window + 1) // 16
        cache.table[i, :gone] = -1
        cache.table[i, :gone:2] = cache.pages - 1 if cache.pages - 1 not in cache.table[i] else -1
    q = torch.randn((cache.tokens, 6, 128), generator=cache.gen).to(BF16)
    P.device_error(lmx)
    got, lse = attend(lmx, cache, q, 6, 0.09, window)
    assert P.device_error(lmx) == 0
    if rows == 0:
        check(cache, q, got, lse, 0.09, window)
    elif bits == 16:
        check(cache, q, got, lse, 0.09, window, p_err=2.0 ** -8)
    else:
        check(cache, q, got, lse, 0.09, window, p_err=2.0 ** -11, kv_err=2.0 ** -11)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_prompt_kernel_unaligned_output_and_far_stride(lmx, cuda, prompt_rows, bits):
    # outputs 16- but not 32-byte aligned take the narrow stores
    prompt_rows(1)
    cache = P.Cache(19, [(100, 250), (1, 3)], 1, 64, bits, 64)
    kv, batch = cache.device(lmx)
    q = torch.randn((101, 4, 64), generator=cache.gen).to(BF16)
    dq = q.cuda()
    size = lmx.lib().lmx_paged_attention_scratch_bytes(kv, batch, 4)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    res = []
    for off, ld in ((0, 256), (8, 264)):
        out = torch.full((102 * 264,), 9.0, dtype=BF16, device="cuda")
        lmx.call("lmx_paged_attention", kv, batch, dq.data_ptr(), 256, 4, 0.125, 0, scratch.data_ptr(), size,
                 out.data_ptr() + 2 * off, ld, None, None)
        res.append(out[off:off + 101 * ld].view(101, ld)[:, :256].clone())
        assert (out[:off] == 9.0).all() and (out[off + 101 * ld:] == 9.0).all()
    assert torch.equal(res[0], res[1])


def test_attention_missing_page_reads_zeros(lmx, cuda):
    cache = P.Cache(15, [(1, 50)], 1, 64, 16, 16)
    cache.table[0, 1] = cache.pages + 5
    for m in "kv":
        cache.rows[m][0][16:32] = 0
    q = torch.randn((1, 4, 64), generator=cache.gen).to(BF16)
    P.device_error(lmx)
    got, lse = attend(lmx, cache, q, 4, 0.125, 0)
    assert P.device_error(lmx) == 0x44
    check(cache, q, got, lse, 0.125, 0)


def test_attention_rows_past_the_table(lmx, cuda):
    # kv_len beyond the table: what the table covers is attended, and the error word says so
    cache = P.Cache(16, [(1, 32)], 1, 64, 16, 16, spare=0)
    kv, batch = cache.device(lmx)
    cache.index[1].fill_(40)
    q = torch.randn((1, 2, 64), generator=cache.gen).to(BF16)
    dq, out = q.cuda(), torch.empty((1, 2, 64), dtype=BF16, device="cuda")
    size = lmx.lib().lmx_paged_attention_scratch_bytes(kv, batch, 2)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    P.device_error(lmx)
    args = [kv, batch, dq.data_ptr(), 128, 2, 0.125, 0, scratch.data_ptr(), size, out.data_ptr(), 128, None, None]
    lmx.call("lmx_paged_attention", *args)
    torch.cuda.synchronize()
    assert P.device_error(lmx) == 0x44
    want, _, A, Q = P.attention(cache, q, 0.125, 0)
    assert ((out.cpu().double() - want).abs() <= U * want.abs() + A * 2.0 ** -12).all()
    # and the host's own checks, which need the scratch size
    args[8] = size - 1
    assert lmx.lib().lmx_paged_attention(*args) == 1 and b"scratch" in lmx.lib().lmx_last_error()
    args[8], args[6] = size, -1
    assert lmx.lib().lmx_paged_attention(*args) == 1
    args[6], args[3] = 0, 120
    assert lmx.lib().lmx_paged_attention(*args) == 1
    for scale in (0.0, -1.0, math.nan, math.inf):
        args[3], args[5] = 128, scale
        assert lmx.lib().lmx_paged_attention(*args) == 1
