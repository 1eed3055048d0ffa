"""The rotary and paged-cache entry points refuse bad arguments with a status
and a message before any device work (so this runs without a GPU)."""
import pytest

OK, INVALID, UNSUPPORTED = 0, 1, 2
A = 4096  # an aligned address that is never read


def kv(lmx, **over):
    f = dict(pages=4, page_size=32, kv_heads=2, head_dim=128, bits=16, page_stride=0, k=A, v=A)
    f.update(over)
    return lmx.PagedKvDesc(**f)


def q4(lmx, **over):
    f = dict(bits=4, k=None, v=None, k_packed=A, v_packed=A, k_scales=A, k_biases=A, v_scales=A, v_biases=A)
    f.update(over)
    return kv(lmx, **f)


def batch(lmx, **over):
    f = dict(seqs=1, tokens=3, max_new=3, q_start=A, kv_len=A, block_table=A, table_stride=2)
    f.update(over)
    return lmx.PagedBatch(**f)


BAD_KV = [(dict(bits=5), UNSUPPORTED), (dict(head_dim=96), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED),
          (dict(page_size=8), UNSUPPORTED), (dict(page_size=512), UNSUPPORTED), (dict(pages=0), INVALID),
          (dict(kv_heads=0), INVALID), (dict(page_stride=63), INVALID), (dict(k=None), INVALID),
          (dict(v=A + 8), INVALID)]
BAD_Q4 = [(dict(page_stride=70), INVALID), (dict(k_packed=None), INVALID), (dict(v_biases=None), INVALID),
          (dict(k_scales=A + 2), INVALID)]
BAD_BATCH = [(dict(seqs=-1), INVALID), (dict(tokens=-1), INVALID), (dict(max_new=-1), INVALID),
             (dict(seqs=2049), UNSUPPORTED), (dict(q_start=None), INVALID), (dict(kv_len=None), INVALID),
             (dict(block_table=None), INVALID), (dict(table_stride=0), INVALID)]


def calls(lmx, cache, b):
    L = lmx.lib()
    return [L.lmx_paged_gather(cache, b, A, A, None),
            L.lmx_paged_append(cache, b, None, None, A, A, 256, 0, None, None, 0.0, None, 0, None),
            L.lmx_paged_attention(cache, b, A, 512, 4, 1.0, 0, A, 1 << 30, A, 512, None, None)]


@pytest.mark.parametrize("over,status", BAD_KV)
def test_bad_cache(lmx, over, status):
    assert calls(lmx, kv(lmx, **over), batch(lmx)) == [status] * 3
    assert lmx.lib().lmx_paged_attention_scratch_bytes(kv(lmx, **over), batch(lmx), 4) == 0
    assert b"paged_attention" in lmx.lib().lmx_last_error()


@pytest.mark.parametrize("over,status", BAD_Q4)
def test_bad_quantized_cache(lmx, over, status):
    assert calls(lmx, q4(lmx, **over), batch(lmx)) == [status] * 3


@pytest.mark.parametrize("over,status", BAD_BATCH)
def test_bad_batch(lmx, over, status):
    assert calls(lmx, kv(lmx), batch(lmx, **over)) == [status] * 3


def test_null_descriptors(lmx):
    assert calls(lmx, None, batch(lmx)) == [INVALID] * 3
    assert calls(lmx, kv(lmx), None) == [INVALID] * 3


def test_nothing_to_do(lmx):
    L, b = lmx.lib(), batch(lmx, tokens=0, seqs=0, q_start=None, kv_len=None, block_table=None, table_stride=0)
    assert L.lmx_paged_gather(kv(lmx), b, A, A, None) == OK
    assert L.lmx_paged_append(kv(lmx), b, None, None, A, A, 256, 0, None, None, 0.0, None, 0, None) == OK
    r = lmx.RopeDesc(A, A, 10, 64, 0)
    assert L.lmx_rope_apply(r, A, 256, A, 0, 2, 128, 0, A, 256, None) == OK


# heads, ldq, ldo, q, out, window
@pytest.mark.parametrize("heads,ldq,ldo,q,out,window,status", [
    (3, 512, 512, A, A, 0, UNSUPPORTED), (0, 512, 512, A, A, 0, UNSUPPORTED), (130, 1 << 20, 1 << 20, A, A, 0, UNSUPPORTED)])
def test_bad_attention(lmx, heads, ldq, ldo, q, out, window, status):
    rc = lmx.lib().lmx_paged_attention(kv(lmx), batch(lmx), q, ldq, heads, 1.0, window, A, 1 << 30, out, ldo, None, None)
    assert rc == status


@pytest.mark.parametrize("args", [
    # q, k, v, ld, heads, q_norm, k_norm, q_out, ldq_out
    (A, A, A, 1024, 4, None, None, None, 0),         # q without q_out
    (A, A, A, 1024, 0, None, None, A, 512),          # no heads
    (A, A, A, 504, 4, None, None, A, 512),           # rows too narrow
    (A, A, A, 1028, 4, None, None, A, 512),          # rows off alignment
    (A, A, A, 1024, 4, None, None, A, 504),
    (A, A, A, 1024, 4, None, None, A, 512),          # in place with another distance
    (A, None, A, 1024, 4, None, None, A + 1024, 512),
    (A, A, A + 2, 1024, 4, None, None, A + 1024, 512),
    (A, A, A, 1024, 4, A, None, A + 1024, 512),      # one norm
    (A, A, A, 1024, -1, None, None, A + 1024, 512),
])
def test_bad_append(lmx, args):
    q, k, v, ld, heads, qn, kn, qo, ldqo = args
    assert lmx.lib().lmx_paged_append(kv(lmx), batch(lmx), None, q, k, v, ld, heads, qn, kn, 1e-6, qo, ldqo, None) == INVALID


@pytest.mark.parametrize("rope", [(None, A, 10, 64, 0), (A, A + 4, 10, 64, 0), (A, A, 0, 64, 0), (A, A, 10, 72, 0),
                                  (A, A, 10, 144, 0), (A, A, 10, 0, 0)])
def test_bad_rope_tables(lmx, rope):
    L, r = lmx.lib(), lmx.RopeDesc(*rope)
    assert L.lmx_rope_apply(r, A, 256, A, 1, 2, 128, 0, A, 256, None) == INVALID
    assert L.lmx_paged_append(kv(lmx), batch(lmx), r, None, A, A, 256, 0, None, None, 0.0, None, 0, None) == INVALID


@pytest.mark.parametrize("args", [
    # x, ldx, pos, tokens, heads, head_dim, y, ldy
    (None, 256, A, 1, 2, 128, A, 256), (A, 256, None, 1, 2, 128, A, 256), (A, 248, A, 1, 2, 128, A, 256),
    (A, 260, A, 1, 2, 128, A + 512, 256), (A, 264, A, 1, 2, 128, A, 256), (A, 256, A, -1, 2, 128, A, 256),
    (A, 256, A, 1, -2, 128, A, 256), (A, 256, A, 1, 2, 120, A, 256), (A, 1024, A, 1, 2, 272, A, 1024)])
def test_bad_rope_rows(lmx, args):
    x, ldx, pos, tokens, heads, dim, y, ldy = args
    r = lmx.RopeDesc(A, A, 10, 64, 0)
    assert lmx.lib().lmx_rope_apply(r, x, ldx, pos, tokens, heads, dim, 0, y, ldy, None) == INVALID


@pytest.mark.parametrize("scaling,positions,rot,status", [
    ((7, 1e4, 1, 0, 0, 0, 0), 8, 64, UNSUPPORTED), ((0, 0.0, 1, 0, 0, 0, 0), 8, 64, INVALID),
    ((0, 1e4, 1, 0, 0, 0, 0), 0, 64, INVALID), ((0, 1e4, 1, 0, 0, 0, 0), 8, 40, INVALID),
    ((0, 1e4, 1, 0, 0, 0, 0), 8, 272, INVALID), ((0, 1e4, 1, 0, 0, 0, 0), 1 << 30, 64, INVALID),
    ((1, 1e4, 0.5, 0, 0, 0, 0), 8, 64, INVALID), ((2, 1e4, 8, 4, 1, 8192, 0), 8, 64, INVALID),
    ((3, 1e4, 8, 1, 32, 0, 0), 8, 64, INVALID), ((3, 0.5, 8, 1, 32, 4096, 0), 8, 64, INVALID)])
def test_bad_rope_scaling(lmx, scaling, positions, rot, status):
    assert lmx.lib().lmx_rope_table(lmx.RopeScaling(*scaling), positions, rot, A, A, None) == status
    assert b"rope_table" in lmx.lib().lmx_last_error()
