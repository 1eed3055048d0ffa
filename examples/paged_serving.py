"""Continuous batching over a paged KV cache.

Requests of unequal lengths share one pool of pages.  Every step packs what
each running request has to compute -- a chunk of its prompt, or its last
token -- into one batch and runs the decoder once:

  projection (lmx_quantized_matmul) -> lmx_paged_append (q / k norm, rotary
  positions, rows into the pages) -> lmx_paged_attention -> projection ...

A request that ends returns its pages; the next one takes them.  The decoder is
a seeded Qwen3 / Llama model of this library whose packed weights are read back
once (lmx_model_weight).  Needs a B200 and torch (device buffers, and the
elementwise glue: embedding, residual, SwiGLU).

    python examples/paged_serving.py
"""
import ctypes as C
import importlib.util
import os

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16 = torch.bfloat16


def load_lmx():
    spec = importlib.util.spec_from_file_location("lmx", os.path.join(ROOT, "lemon-mlx-engine_b200", "lmx.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def device_weight(lmx, model, layer, kind, rows, cols, bits):
    w = np.zeros((rows, cols * bits // 32), np.uint32)
    s, b = (np.zeros((rows, cols // 64), np.uint16) for _ in "sb")
    lmx.call("lmx_model_weight", model.h, layer, kind, w.ctypes.data, s.ctypes.data, b.ctypes.data)
    return (torch.from_numpy(w.view(np.int32)).cuda(),) + tuple(torch.from_numpy(x.view(np.int16)).cuda().view(BF16)
                                                                for x in (s, b))


class Pages:
    """The pool: one cache per layer, one free list for all of them."""

    def __init__(self, lmx, cfg, pages, page_size, bits):
        self.size, self.bits, self.free = page_size, bits, list(range(pages))
        hk, d = cfg["kv_heads"], cfg["head_dim"]
        shape = (pages, hk, page_size)
        self.layers, self.keep = [], []
        for _ in range(cfg["layers"]):
            if bits == 16:
                t = [torch.empty(shape + (d,), dtype=BF16, device="cuda") for _ in "kv"]
                f = [x.data_ptr() for x in t]
            else:
                t = [torch.empty(shape + (d * bits // 8,), dtype=torch.uint8, device="cuda") for _ in "kv"]
                t += [torch.empty(shape + (d // 64,), dtype=BF16, device="cuda") for _ in range(4)]
                f = [None, None] + [x.data_ptr() for x in t]
            self.layers.append(lmx.PagedKvDesc(pages, page_size, hk, d, bits, 0, *f))
            self.keep += t


class Request:
    def __init__(self, prompt, max_tokens):
        self.prompt, self.max_tokens = list(prompt), max_tokens
        self.done, self.tokens, self.pages = 0, [], []  # rows cached, tokens generated, pages held

    def pending(self, chunk):
        """The tokens of this request in the next step."""
        seq = self.prompt + self.tokens
        return seq[self.done:self.done + chunk]

    def finished(self):
        return len(self.tokens) >= self.max_tokens


class Server:
    def __init__(self, lmx, cfg, seed, pages=256, page_size=32, kv_bits=16, positions=4096, chunk=128):
        self.lmx, self.cfg, self.chunk = lmx, cfg, chunk
        model = lmx.Model(cfg, seed)
        H, D, bits, I = cfg["hidden"], cfg["head_dim"], cfg["bits"], cfg["inter"]
        nq, nk = cfg["heads"] * D, cfg["kv_heads"] * D
        shapes = [(nq, H), (nk, H), (nk, H), (H, nq), (I, H), (I, H), (H, I)]
        self.w = []
        for l in range(cfg["layers"]):
            q, k, v, o, g, u, dn = (device_weight(lmx, model, l, i, r, c, bits) for i, (r, c) in enumerate(shapes))
            # q | k | v and gate | up as one projection each
            self.w.append([tuple(torch.cat(x).contiguous() for x in zip(q, k, v)), o,
                           tuple(torch.cat(x).contiguous() for x in zip(g, u)), dn])
        e = device_weight(lmx, model, 0, 7, cfg["vocab"], H, bits)
        self.head = e if cfg["tied"] else device_weight(lmx, model, 0, 8, cfg["vocab"], H, bits)
        codes = e[0].view(torch.uint8)
        codes = codes if bits == 8 else torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
        self.embed = (codes.float().unflatten(-1, (-1, 64)) * e[1].float()[..., None] + e[2].float()[..., None]).flatten(-2).to(BF16)
        model.close()
        self.ones = {n: torch.ones(n, dtype=BF16, device="cuda") for n in (H, D)}  # seeded models' norm weights
        self.cos, self.sin = (torch.empty(positions, D // 2, device="cuda") for _ in "cs")
        scaled = cfg.get("rope_factor", 0.0) > 1.0
        lmx.call("lmx_rope_table",
                 lmx.RopeScaling(lmx.ROPE_LLAMA3 if scaled else lmx.ROPE_PLAIN, cfg["rope_theta"], cfg.get("rope_factor", 1.0),
                                 cfg.get("rope_low_freq", 1.0), cfg.get("rope_high_freq", 4.0),
                                 cfg.get("rope_orig_max_pos", 8192.0), 0.0),
                 positions, D, self.cos.data_ptr(), self.sin.data_ptr(), None)
        self.rope = lmx.RopeDesc(self.cos.data_ptr(), self.sin.data_ptr(), positions, D, 0)
        self.pages = Pages(lmx, cfg, pages, page_size, kv_bits)
        self.scratch = torch.empty(0, dtype=torch.uint8, device="cuda")

    def matmul(self, x, w):
        y = torch.empty((x.shape[0], w[0].shape[0]), dtype=BF16, device="cuda")
        self.lmx.call("lmx_quantized_matmul", x.data_ptr(), w[0].data_ptr(), w[1].data_ptr(), w[2].data_ptr(), y.data_ptr(),
                      x.shape[0], w[0].shape[0], x.shape[1], 64, self.cfg["bits"], None)
        return y

    def norm(self, x):
        y = torch.empty_like(x)
        self.lmx.call("lmx_rms_norm", x.data_ptr(), self.ones[x.shape[1]].data_ptr(), y.data_ptr(), x.shape[0], x.shape[1],
                      self.cfg["eps"], None)
        return y

    def step(self, requests):
        """One batch of every request's pending tokens.  Returns each request's last logits [n, vocab]; a request whose
        prompt is through gets its next (greedy) token."""
        lmx, cfg = self.lmx, self.cfg
        new = [r.pending(self.chunk) for r in requests]
        for r, t in zip(requests, new):
            while len(r.pages) * self.pages.size < r.done + len(t):
                r.pages.append(self.pages.free.pop())
        start = np.concatenate([[0], np.cumsum([len(t) for t in new])]).astype(np.int32)
        length = np.array([r.done + len(t) for r, t in zip(requests, new)], np.int32)
        table = np.zeros((len(requests), max(len(r.pages) for r in requests)), np.int32)
        for i, r in enumerate(requests):
            table[i, :len(r.pages)] = r.pages
        d_start, d_len, d_table = (torch.from_numpy(a).cuda() for a in (start, length, table))
        n, Hq, Hk, D = int(start[-1]), cfg["heads"], cfg["kv_heads"], cfg["head_dim"]
        batch = lmx.PagedBatch(len(requests), n, max(len(t) for t in new), d_start.data_ptr(), d_len.data_ptr(),
                               d_table.data_ptr(), table.shape[1])
        need = lmx.lib().lmx_paged_attention_scratch_bytes(self.pages.layers[0], batch, Hq)
        if need > self.scratch.numel():
            self.scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
        norm = self.ones[D].data_ptr() if cfg["qk_norm"] else None

        h = self.embed[torch.tensor(np.concatenate(new), dtype=torch.long, device="cuda")]
        for (qkv_w, o_w, gu_w, d_w), kv in zip(self.w, self.pages.layers):
            qkv = self.matmul(self.norm(h), qkv_w)
            p, ld = qkv.data_ptr(), qkv.shape[1]
            # q is rotated in place; k and v go to their pages
            lmx.call("lmx_paged_append", kv, batch, self.rope, p, p + 2 * Hq * D, p + 2 * (Hq + Hk) * D, ld, Hq, norm, norm,
                     cfg["eps"], p, ld, None)
            att = torch.empty((n, Hq * D), dtype=BF16, device="cuda")
            lmx.call("lmx_paged_attention", kv, batch, p, ld, Hq, D ** -0.5, 0, self.scratch.data_ptr(), self.scratch.numel(),
                     att.data_ptr(), Hq * D, None, None)
            h = h + self.matmul(att, o_w)
            g, u = self.matmul(self.norm(h), gu_w).chunk(2, -1)
            h = h + self.matmul(torch.nn.functional.silu(g) * u, d_w)
        last = torch.from_numpy(start[1:] - 1).long().cuda()
        logits = self.matmul(self.norm(h)[last].contiguous(), self.head)
        pick = torch.empty(len(requests), dtype=torch.int32, device="cuda")
        lmx.call("lmx_argmax", logits.data_ptr(), len(requests), cfg["vocab"], pick.data_ptr(), None)
        for r, t, tok in zip(requests, new, pick.tolist()):
            r.done += len(t)
            if r.done == len(r.prompt) + len(r.tokens):
                r.tokens.append(tok)
        return logits

    def serve(self, requests, most=8):
        """Run all requests, at most `most` at a time, in order of arrival."""
        waiting, running = list(requests), []
        while waiting or running:
            while waiting and len(running) < most:
                running.append(waiting.pop(0))
            self.step(running)
            for r in [r for r in running if r.finished()]:
                self.pages.free += r.pages
                r.pages = []
                running.remove(r)
        err = C.c_uint(0)
        self.lmx.call("lmx_device_error", C.byref(err), 1)
        if err.value:
            raise self.lmx.LmxError(f"device error 0x{err.value:x}")
        return requests


def main():
    lmx = load_lmx()
    cfg = dict(hidden=1024, layers=4, inter=2048, heads=16, kv_heads=8, head_dim=128, vocab=4000, rope_theta=1e6, eps=1e-6,
               qk_norm=1, tied=1, bits=4, group_size=64)
    rng = np.random.RandomState(0)
    requests = [Request(rng.randint(0, cfg["vocab"], n), m) for n, m in ((300, 24), (5, 40), (77, 8), (1, 30), (512, 12), (140, 20))]
    server = Server(lmx, cfg, 7, kv_bits=8)
    server.serve(requests, most=4)
    for i, r in enumerate(requests):
        print(f"request {i}: prompt {len(r.prompt)}, {len(r.tokens)} tokens: {r.tokens[:8]} ...")
    print(f"{len(server.pages.free)} pages free again")


if __name__ == "__main__":
    main()
