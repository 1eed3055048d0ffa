"""Timed cases of the paged-cache operators: rotary positions, appending to a
paged key / value cache (with the rotation and the cache's quantizer on the
way) and attention of new tokens over the paged cache.

Each case runs in a plain form (elementary torch operations in 32 bits,
rounded once) or, with `own`, through the library's entry points.  A cache
page holds `page` rows of every KV head, [pages][kv_heads][page][head_dim];
4- and 8-bit caches keep affine codes with one bf16 scale and bias per 64
values.  The new tokens of all sequences are packed one after another."""
import importlib.util
import math
import os
import random

import torch

own = False

GROUP = 64
EPS = 1e-6
POSITIONS = 16640  # rows of the rotation tables (the longest context and its new tokens)
BF16 = torch.bfloat16


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def _rope(name, tokens, heads, dim, rot, interleaved, scaling, inverse=False):
    return dict(name=name, op="rope", tokens=tokens, heads=heads, dim=dim, rot=rot, interleaved=interleaved,
                scaling=scaling, inverse=inverse)


def _append(name, seqs, new, ctx, mode, heads, kv_heads, dim, bits, page, rot, interleaved, scaling, norm, mix):
    return dict(name=name, op="append", seqs=seqs, new=new, ctx=ctx, mode=mode, heads=heads, kv_heads=kv_heads,
                dim=dim, bits=bits, page=page, rot=rot, interleaved=interleaved, scaling=scaling, norm=norm, mix=mix)


def _attend(name, seqs, new, ctx, mode, heads, kv_heads, dim, bits, page, window, lse, mix):
    return dict(name=name, op="attend", seqs=seqs, new=new, ctx=ctx, mode=mode, heads=heads, kv_heads=kv_heads,
                dim=dim, bits=bits, page=page, window=window, lse=lse, mix=mix)


def listed():
    return [
        # one decode step of the 0.6B draft for 8 sequences: its q and k heads inside the fused q|k|v rows
        _rope("rope_tokens", 8, 24, 128, 128, False, "none"),
        # a long prompt, half of each head rotated in interleaved pairs, positions stretched for a long context
        _rope("rope_prompt", 8191, 40, 128, 64, True, "yarn"),
        # one decode step of 32 requests, 64-wide heads, small pages
        _append("append_tokens", 32, 1, 2000, "same", 32, 8, 64, 16, 16, 64, False, "llama3", False, 1),
        # ragged prompt chunks of an 8B model with q / k norms into a bf16 cache
        _append("append_chunks", 5, 2048, 3000, "ragged", 32, 8, 128, 16, 64, 128, False, "none", True, 2),
        # prompts of a 70B model into a 4-bit cache, and the rows read back
        _append("append_chunks_4bit", 3, 4096, 4000, "ragged", 64, 8, 128, 4, 128, 128, False, "linear", False, 3),
        # five verify tokens of 16 sequences into an 8-bit cache at a long context, and the rows read back
        _append("append_verify_8bit", 16, 5, 8192, "same", 64, 8, 128, 8, 32, 128, False, "none", False, 4),
        # the smallest call: one token of one request, short context
        _attend("attend_token", 1, 1, 700, "same", 16, 8, 128, 16, 16, 0, True, 5),
        # one decode step of 16 requests at a long context, 8-bit cache
        _attend("attend_tokens_8bit", 16, 1, 8192, "same", 64, 8, 128, 8, 64, 0, False, 6),
        # the verify pass of 5 drafts for 8 requests over a 4-bit cache
        _attend("attend_verify_4bit", 8, 6, 1024, "same", 32, 8, 128, 4, 32, 0, False, 7),
        # decode tokens and prompt chunks in one batch, sliding window, three query heads per KV head
        _attend("attend_mixed_window", 24, 512, 4096, "mixed", 24, 8, 128, 8, 64, 1024, False, 8),
        # whole ragged prompts from an empty cache, 64-wide heads
        _attend("attend_prompts_64", 5, 4000, 0, "ragged", 32, 8, 64, 16, 16, 0, True, 9),
        # the largest: one 8192-token prompt of the 70B model
        _attend("attend_prompt", 1, 8192, 0, "same", 64, 8, 128, 16, 128, 0, False, 10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    scaling = rng.choice(["none", "linear", "llama3", "yarn"])
    dim = rng.choice([64, 128, 128])
    rot = rng.choice([dim, dim, dim // 2])
    interleaved = rng.random() < 0.4
    bits = rng.choice([16, 16, 8, 4])
    page = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    mix = rng.randrange(1 << 20)
    op = rng.choice(["rope", "append", "append", "attend", "attend", "attend", "attend"])
    if op == "rope":
        return _drop(_rope("", _log(rng, 1, 8191), rng.choice([1, 5, 9, 24, 40]), dim, rot, interleaved, scaling,
                           rng.random() < 0.3))
    mode = rng.choice(["same", "ragged", "mixed"])
    while True:
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, 8) if mode == "same" else _log(rng, 2, 4096)
        ctx = _log(rng, 1, 8192)
        longest = ctx + new
        if op == "append":
            if seqs * new * (heads + 2 * kv_heads) * dim <= 1 << 27 and seqs * longest * kv_heads * dim <= 1 << 28:
                return _drop(_append("", seqs, new, ctx, mode, heads, kv_heads, dim, bits, page, rot, interleaved,
                                     scaling, bits == 16 and rng.random() < 0.4, mix))
        elif seqs * heads * new * longest <= 1 << 31 and seqs * longest * kv_heads * dim <= 1 << 27:
            window = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
            return _drop(_attend("", seqs, new, ctx, mode, heads, kv_heads, dim, bits, page, window, bits == 16, mix))


def _drop(case):
    del case["name"]
    return case


def _lengths(case):
    """(new tokens, cached rows before them) of each sequence."""
    rng = random.Random(case["mix"])
    out = []
    for i in range(case["seqs"]):
        new = case["new"]
        if case["mode"] == "ragged":
            new = case["new"] if i == 0 else rng.randint(1, case["new"])
        elif case["mode"] == "mixed":
            new = case["new"] if i == 0 else 1 if rng.random() < 0.7 else rng.randint(1, case["new"])
        ctx = case["ctx"]
        if ctx > 0 and i > 0:
            ctx = rng.randint(ctx // 2, ctx) if case["mode"] == "same" else rng.randint(0, ctx)
        out.append((new, ctx))
    return out


# ---------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------
def _frequencies(rot, scaling):
    """Angular frequencies of the rot/2 pairs (64 bits) and the factor on cos and sin."""
    theta, orig, factor = 500000.0, 8192.0, 8.0
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "llama3":  # wavelengths above the low bound stretched, a ramp in between
        ramp = ((orig * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * (ramp + (1 - ramp) / factor), 1.0
    if scaling == "yarn":  # a ramp over the pair index between 32 and 1 turns in the original context
        at = [rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _tables(rot, scaling):
    f, mul = _frequencies(rot, scaling)
    angle = torch.arange(POSITIONS, dtype=torch.float64)[:, None] * f
    return (angle.cos() * mul).float().cuda(), (angle.sin() * mul).float().cuda()


def _normal(gen, shape, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(BF16)


def _quantize(x, bits):
    """x [..., dim] float -> codes (uint8 values), bf16 scales and biases [..., dim / 64]."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    top = torch.tensor(float((1 << bits) - 1), device=x.device, dtype=x.dtype)
    s = ((hi - lo) / top).to(BF16)
    s = torch.where(s == 0, torch.ones_like(s), s)
    b = lo.to(BF16)
    q = ((g - b.to(x.dtype)[..., None]) / s.to(x.dtype)[..., None]).round().clamp(0, (1 << bits) - 1)
    return q.flatten(-2).to(torch.uint8), s, b


def _pack(q, bits):
    return q if bits == 8 else (q[..., 0::2] | (q[..., 1::2] << 4))


def _values(packed, s, b, bits):
    """The values that codes stand for, in 32 bits."""
    q = packed if bits == 8 else torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    g = q.float().unflatten(-1, (-1, GROUP))
    return (g * s.float()[..., None] + b.float()[..., None]).flatten(-2)


def _pool(case, gen, pages):
    """A pool of pages holding earlier rows."""
    shape, st = (pages, case["kv_heads"], case["page"], case["dim"]), {}
    for n in "kv":
        x = _normal(gen, shape)
        if case["bits"] == 16:
            st[n] = x
        else:
            q, s, b = _quantize(x.float(), case["bits"])
            st[n], st[n + "s"], st[n + "b"] = _pack(q, case["bits"]), s, b
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng = random.Random(seed)
    st = dict(case=case)
    if case["op"] == "rope":
        n, h, d = case["tokens"], case["heads"], case["dim"]
        st["cos"], st["sin"] = _tables(case["rot"], case["scaling"])
        row = _normal(gen, (n, h + 8, d))  # q and k heads in front of 8 v heads
        st["x"] = row[:, :h]
        first = rng.randrange(POSITIONS - n)
        st["pos"] = torch.arange(first, first + n, dtype=torch.int32, device="cuda")
        return st
    lens, page = _lengths(case), case["page"]
    new = [n for n, _ in lens]
    total = [n + c for n, c in lens]
    blocks = [-(-t // page) for t in total]
    pages = sum(blocks) + 3
    order = list(range(pages))
    rng.shuffle(order)
    table = torch.zeros(len(lens), max(blocks), dtype=torch.int32)
    for i, n in enumerate(blocks):
        table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    st.update(seqs=len(lens), tokens=start[-1], max_new=max(new), max_len=max(total), pages=pages,
              q_start=torch.tensor(start, dtype=torch.int32, device="cuda"),
              kv_len=torch.tensor(total, dtype=torch.int32, device="cuda"), table=table.cuda())
    st["pool"] = _pool(case, gen, pages)
    h, hk, d, n = case["heads"], case["kv_heads"], case["dim"], start[-1]
    if case["op"] == "append":
        st["cos"], st["sin"] = _tables(case["rot"], case["scaling"])
        row = _normal(gen, (n, h + 2 * hk, d))  # the fused projection's rows
        st["q"], st["k"], st["v"] = row[:, :h], row[:, h:h + hk], row[:, h + hk:]
        if case["norm"]:
            st["qn"], st["kn"] = [(1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(BF16) for _ in "qk"]
    else:
        st["q"] = _normal(gen, (n, h, d), 1.5)
    return st


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _rotate(x, c, s, interleaved):
    """x [tokens, heads, dim] in 32 bits; c, s [tokens, rot / 2]."""
    rot = 2 * c.shape[-1]
    c, s = c[:, None], s[:, None]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_rope(st):
    case, pos = st["case"], st["pos"].long()
    s = st["sin"][pos]
    return {"y": _rotate(st["x"].float(), st["cos"][pos], -s if case["inverse"] else s, case["interleaved"]).to(BF16)}


def _rows(st):
    """Sequence and position of each packed token."""
    t = torch.arange(st["tokens"], device="cuda")
    seq = torch.searchsorted(st["q_start"][1:].long(), t, right=True)
    return seq, st["kv_len"][seq].long() - st["q_start"][seq + 1].long() + t


def _plain_append(st):
    case, pool = st["case"], st["pool"]
    seq, pos = _rows(st)
    page, slot = st["table"][seq, pos // case["page"]].long(), pos % case["page"]
    c, s = st["cos"][pos], st["sin"][pos]
    q, k = st["q"].float(), st["k"].float()
    if case["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * st["qn"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * st["kn"].float()
    out = {"q": _rotate(q, c, s, case["interleaved"]).to(BF16)}
    for n, x in (("k", _rotate(k, c, s, case["interleaved"])), ("v", st["v"].float())):
        if case["bits"] == 16:
            pool[n][page, :, slot] = x.to(BF16)
            out[n] = pool[n]
        else:
            codes, scale, bias = _quantize(x, case["bits"])
            pool[n][page, :, slot] = _pack(codes, case["bits"])
            pool[n + "s"][page, :, slot], pool[n + "b"][page, :, slot] = scale, bias
            out[n] = _values(pool[n][page, :, slot], pool[n + "s"][page, :, slot], pool[n + "b"][page, :, slot],
                             case["bits"]).to(BF16)
    return out


def _plain_attend(st):
    case, pool = st["case"], st["pool"]
    seqs, tm, lm, h, hk, d = st["seqs"], st["max_new"], st["max_len"], case["heads"], case["kv_heads"], case["dim"]
    start, length = st["q_start"].long(), st["kv_len"].long()
    new = start[1:] - start[:-1]
    t = torch.arange(tm, device="cuda")
    j = torch.arange(lm, device="cuda")
    at = (start[:-1, None] + t).clamp(max=st["tokens"] - 1)  # [seqs, tm] rows of q
    q = st["q"][at].float().mul_(1 / math.sqrt(d))
    q = q.view(seqs, tm, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(seqs, hk, -1, d)
    there = j < length[:, None]  # [seqs, lm]
    blocks = st["table"][:, :-(-lm // case["page"])].long()
    kv = {}
    for n in "kv":
        x = pool[n][blocks] if case["bits"] == 16 else _values(pool[n][blocks], pool[n + "s"][blocks],
                                                               pool[n + "b"][blocks], case["bits"])
        x = x.float().transpose(1, 2).flatten(2, 3)[:, :, :lm]  # [seqs, hk, lm, d]
        kv[n] = x * there[:, None, :, None]
    pos = length[:, None] - new[:, None] + t  # [seqs, tm]
    seen = (j <= pos[..., None]) & there[:, None]
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    s = torch.matmul(q, kv["k"].transpose(-1, -2)).view(seqs, hk, h // hk, tm, lm)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, hk, -1, lm), kv["v"]).view(seqs, hk, h // hk, tm, d)
    o = (o / total.clamp(min=1e-30)).permute(0, 3, 1, 2, 4).reshape(seqs, tm, h, d)
    seq, row = _rows(st)
    token = torch.arange(st["tokens"], device="cuda") - start[seq]
    out = {"out": o[seq, token].to(BF16)}
    if case["lse"]:
        out["lse"] = (m + total.log())[..., 0].permute(0, 3, 1, 2).reshape(seqs, tm, h)[seq, token]
    return out


# ---------------------------------------------------------------------------
# The library's operators
# ---------------------------------------------------------------------------
_lmx = None


def _library():
    global _lmx
    if _lmx is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        spec = importlib.util.spec_from_file_location("lmx", os.path.join(root, "lemon-mlx-engine_b200", "lmx.py"))
        _lmx = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_lmx)
    return _lmx


def _own_rope(st, L, stream):
    case, x = st["case"], st["x"]
    y = torch.empty(x.shape, dtype=BF16, device="cuda")
    rope = L.RopeDesc(st["cos"].data_ptr(), st["sin"].data_ptr(), POSITIONS, case["rot"], int(case["interleaved"]))
    L.call("lmx_rope_apply", rope, x.data_ptr(), x.stride(0), st["pos"].data_ptr(), case["tokens"], case["heads"],
           case["dim"], int(case["inverse"]), y.data_ptr(), y.stride(0), stream)
    return {"y": y}


def _own_cache(st, L):
    case, pool = st["case"], st["pool"]
    if case["bits"] == 16:
        kv = L.PagedKvDesc(st["pages"], case["page"], case["kv_heads"], case["dim"], 16, 0, pool["k"].data_ptr(),
                           pool["v"].data_ptr())
    else:
        kv = L.PagedKvDesc(st["pages"], case["page"], case["kv_heads"], case["dim"], case["bits"], 0, None, None,
                           pool["k"].data_ptr(), pool["v"].data_ptr(), pool["ks"].data_ptr(), pool["kb"].data_ptr(),
                           pool["vs"].data_ptr(), pool["vb"].data_ptr())
    batch = L.PagedBatch(st["seqs"], st["tokens"], st["max_new"], st["q_start"].data_ptr(), st["kv_len"].data_ptr(),
                         st["table"].data_ptr(), st["table"].stride(0))
    return kv, batch


def _own_append(st, L, stream):
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    kv, batch = _own_cache(st, L)
    rope = L.RopeDesc(st["cos"].data_ptr(), st["sin"].data_ptr(), POSITIONS, case["rot"], int(case["interleaved"]))
    qo = torch.empty(q.shape, dtype=BF16, device="cuda")
    L.call("lmx_paged_append", kv, batch, rope, q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), case["heads"],
           st["qn"].data_ptr() if case["norm"] else None, st["kn"].data_ptr() if case["norm"] else None, EPS,
           qo.data_ptr(), qo.stride(0), stream)
    if case["bits"] == 16:
        return {"q": qo, "k": st["pool"]["k"], "v": st["pool"]["v"]}
    ko, vo = (torch.empty((st["tokens"], case["kv_heads"], case["dim"]), dtype=BF16, device="cuda") for _ in "kv")
    L.call("lmx_paged_gather", kv, batch, ko.data_ptr(), vo.data_ptr(), stream)
    return {"q": qo, "k": ko, "v": vo}


def _own_attend(st, L, stream):
    case, q = st["case"], st["q"]
    kv, batch = _own_cache(st, L)
    if "scratch" not in st:  # a program keeps its workspace
        st["scratch"] = torch.empty(L.lib().lmx_paged_attention_scratch_bytes(kv, batch, case["heads"]),
                                    dtype=torch.uint8, device="cuda")
    out = torch.empty(q.shape, dtype=BF16, device="cuda")
    lse = torch.empty(q.shape[:2], device="cuda") if case["lse"] else None
    L.call("lmx_paged_attention", kv, batch, q.data_ptr(), q.stride(0), case["heads"], 1 / math.sqrt(case["dim"]),
           case["window"], st["scratch"].data_ptr(), st["scratch"].numel(), out.data_ptr(), out.stride(0),
           lse.data_ptr() if case["lse"] else None, stream)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def run(state):
    op = state["case"]["op"]
    if own:
        L, stream = _library(), torch.cuda.current_stream().cuda_stream
        return {"rope": _own_rope, "append": _own_append, "attend": _own_attend}[op](state, L, stream)
    return {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}[op](state)


# ---------------------------------------------------------------------------
# What each case cannot do without, and its values in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "rope":
        n, h, d, rot = case["tokens"], case["heads"], case["dim"], case["rot"]
        return {"bytes": n * (4 * h * d + 4 * rot + 4), "flops": 3 * n * h * rot}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    row = 2 * d if case["bits"] == 16 else d * case["bits"] // 8 + 4 * d // GROUP  # one head's row of K or V
    lens = _lengths(case)
    if case["op"] == "append":
        n = sum(new for new, _ in lens)
        back = 0 if case["bits"] == 16 else 2 * hk * (row + 2 * d)  # the rows read back
        return {"bytes": n * (4 * h * d + 2 * hk * (2 * d + row) + 4 * case["rot"] + back),
                "flops": n * (3 * (h + hk) * case["rot"] + (4 * (h + hk) * d if case["norm"] else 0)
                              + (0 if case["bits"] == 16 else 8 * hk * d))}
    n = pairs = rows = 0
    for new, ctx in lens:
        w = case["window"] or ctx + new
        full = max(0, min(new, ctx + new - w))  # queries that see a whole window
        part = new - full
        pairs += full * w + part * (2 * ctx + part + 1) // 2
        rows += min(ctx + new, w + new - 1)
        n += new
    return {"bytes": 4 * n * h * d + 2 * hk * rows * row + (4 * n * h if case["lse"] else 0),
            "flops": 4 * h * d * pairs}


def _turn(x, angle, mul, interleaved):
    """x [tokens, heads, dim] as complex pairs turned by angle [tokens, rot / 2]."""
    rot = 2 * angle.shape[-1]
    part = x[..., :rot]
    pairs = part.unflatten(-1, (-1, 2)) if interleaved else part.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.full_like(angle, mul), angle)[:, None]
    y = torch.view_as_real(z)
    y = y.flatten(-2) if interleaved else y.transpose(-1, -2).flatten(-2)
    return torch.cat((y, x[..., rot:]), -1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        f, mul = _frequencies(case["rot"], case["scaling"])
        angle = st["pos"].double()[:, None] * f.cuda()
        return {"y": _turn(st["x"].double(), -angle if case["inverse"] else angle, mul, case["interleaved"])}
    lens, pool, page, d = _lengths(case), st["pool"], case["page"], case["dim"]
    table = st["table"].cpu().tolist()
    if case["op"] == "append":
        f, mul = _frequencies(case["rot"], case["scaling"])
        pos = torch.cat([torch.arange(c, c + n, dtype=torch.float64) for n, c in lens]).cuda()
        q, k, v = (st[n].double() for n in "qkv")
        if case["norm"]:
            q, k = (x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt() * st[w].double()
                    for x, w in ((q, "qn"), (k, "kn")))
        q, k = (_turn(x, pos[:, None] * f.cuda(), mul, case["interleaved"]) for x in (q, k))
        if case["bits"] == 16:
            out = {"q": q, "k": pool["k"].double(), "v": pool["v"].double()}
            where = [(table[i][p // page], p % page) for i, (n, c) in enumerate(lens) for p in range(c, c + n)]
            at = torch.tensor(where, device="cuda")
            out["k"][at[:, 0], :, at[:, 1]], out["v"][at[:, 0], :, at[:, 1]] = k, v
            return out
        out = {"q": q}
        for n, x in (("k", k), ("v", v)):
            g = x.view(x.shape[0], x.shape[1], -1, GROUP)
            low, top = g.min(-1).values, (1 << case["bits"]) - 1
            s, b = ((g.max(-1).values - low) / top).to(BF16).double(), low.to(BF16).double()
            s = torch.where(s > 0, s, torch.ones_like(s))
            out[n] = (torch.clamp(torch.round((g - b[..., None]) / s[..., None]), 0, top) * s[..., None]
                      + b[..., None]).view(x.shape)
        return out
    h, hk = case["heads"], case["kv_heads"]
    out = torch.zeros(st["tokens"], h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((st["tokens"], h), -math.inf, dtype=torch.float64, device="cuda")
    first = 0
    for i, (new, ctx) in enumerate(lens):
        ids = torch.tensor(table[i][:-(-(ctx + new) // page)], device="cuda")
        at = torch.arange(ctx, ctx + new, device="cuda")[:, None]
        j = torch.arange(ctx + new, device="cuda")[None]
        hidden = (j > at) | (j <= at - case["window"]) if case["window"] else j > at
        for g in range(hk):
            kv = []
            for n in "kv":
                x = pool[n][ids, g]
                if case["bits"] != 16:
                    c = x if case["bits"] == 8 else torch.stack((x % 16, x // 16), -1).flatten(-2)
                    s, b = (pool[n + w][ids, g].double().repeat_interleave(GROUP, -1) for w in "sb")
                    x = c.double() * s + b
                kv.append(x.double().flatten(0, 1)[:ctx + new])
            for r in range(g * (h // hk), (g + 1) * (h // hk)):
                z = (st["q"][first:first + new, r].double() @ kv[0].T) / math.sqrt(d)
                z = z.masked_fill(hidden, -math.inf)
                lse[first:first + new, r] = torch.logsumexp(z, -1)
                out[first:first + new, r] = torch.softmax(z, -1) @ kv[1]
        first += new
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
