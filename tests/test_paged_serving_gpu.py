"""examples/paged_serving.py: rotary tables, paged append and paged attention in
a decoder, requests of unequal lengths batched together, against the engine's
own contiguous-cache forward of the same model and tokens."""
import ctypes as C
import importlib.util
import os

import numpy as np
import pytest

import oracle_lib as O

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

QWEN = dict(hidden=512, layers=2, inter=1024, heads=8, kv_heads=2, head_dim=128, vocab=1000, rope_theta=1e6, eps=1e-6,
            qk_norm=1, tied=1, bits=4, group_size=64)
LLAMA = dict(QWEN, qk_norm=0, tied=0, bits=8, rope_theta=5e5, rope_factor=32.0, rope_low_freq=1.0, rope_high_freq=4.0,
             rope_orig_max_pos=64.0)


def example():
    spec = importlib.util.spec_from_file_location("paged_serving", os.path.join(ROOT, "examples", "paged_serving.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("cfg,kv_bits", [(QWEN, 16), (LLAMA, 16), (QWEN, 8)])
def test_batched_requests_match_the_engine(lmx, cuda, cfg, kv_bits):
    ex = example()
    rng = np.random.RandomState(3)
    sv = ex.Server(lmx, cfg, 21, pages=40, page_size=16, kv_bits=kv_bits, positions=512, chunk=64)
    reqs = [ex.Request(rng.randint(0, cfg["vocab"], n), 6) for n in (150, 3, 64)]
    model = lmx.Model(cfg, 21)
    caches = []
    for _ in reqs:
        c = C.c_void_p()
        lmx.call("lmx_cache_create", model.h, cfg["layers"], 1, 200, kv_bits, 64, C.byref(c))
        caches.append(c)
    steps = 0
    while any(not r.finished() for r in reqs):
        live = [i for i, r in enumerate(reqs) if not r.finished()]
        new = [np.array(reqs[i].pending(sv.chunk), np.int32) for i in live]
        got = O.bf16_to_f32(sv.step([reqs[i] for i in live]).view(cuda.int16).cpu().numpy().view(np.uint16))
        for i, tok, g in zip(live, new, got):
            out = np.zeros((1, len(tok), cfg["vocab"]), np.uint16)
            lmx.call("lmx_forward", model.h, caches[i], cfg["layers"], tok.ctypes.data, 1, len(tok), out.ctypes.data)
            ref = O.bf16_to_f32(out[0, -1])
            # the two paths round at other places (bf16 residuals and SwiGLU alike, attention and q / k norms
            # not): the engine's own tolerance between its paths, 4e-2 and a bf16 ulp (1e-1 over a quantized
            # cache, where a code may move by a step), and the picks agree where the ranking is clear
            lim = (4e-2 if kv_bits == 16 else 1e-1) + np.abs(ref) * 2.0 ** -7
            assert (np.abs(g - ref) <= lim).all(), (steps, i, np.abs(g - ref).max())
            top = np.sort(ref)[-2:]
            if top[1] - top[0] > 2 * lim.max():
                assert g.argmax() == ref.argmax()
        steps += 1
    assert steps == 3 + 5  # three prompt chunks of the longest, then its tokens
    for c in caches:
        lmx.call("lmx_cache_free", c)
    model.close()


def test_pages_are_shared_and_returned(lmx, cuda):
    ex = example()
    rng = np.random.RandomState(4)
    prompts = [rng.randint(0, QWEN["vocab"], n) for n in (70, 1, 33, 90, 16)]
    alone = []
    for p in prompts:  # each request by itself
        sv = ex.Server(lmx, QWEN, 5, pages=16, page_size=16, positions=256, chunk=32)
        alone.append(sv.serve([ex.Request(p, 5)])[0].tokens)
    sv = ex.Server(lmx, QWEN, 5, pages=16, page_size=16, positions=256, chunk=32)
    reqs = sv.serve([ex.Request(p, 5) for p in prompts], most=3)
    assert sorted(sv.pages.free) == list(range(16))
    assert [len(r.tokens) for r in reqs] == [5] * 5
    # another batch gives other matmul shapes: most streams agree token for token, and all begin alike where the
    # first pick is clear
    assert sum(a == r.tokens for a, r in zip(alone, reqs)) >= 3
