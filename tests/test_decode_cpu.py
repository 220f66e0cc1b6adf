"""CPU: what the attention decoder's entry points refuse, before any device
work, and the sizes that they ask for."""
import ctypes

import pytest

P = 1 << 20  # a pointer that is aligned and never followed: every call here is refused before


def cache(**kw):
    import pkc
    a = dict(k=P, v=P, k_scale=P, v_scale=P, table=P, n_pages=8, page=16, n_kv_heads=2, head_dim=64, table_ld=4)
    a.update(kw)
    return pkc.KV8Cache(**a)


def refused(fn, *args, **kw):
    import pkc
    with pytest.raises(pkc.PkcError) as e:
        fn(*args, **kw)
    assert e.value.status == pkc.PKC_ERR_ARG, e.value
    return str(e.value)


def cross(**kw):
    import pkc
    a = dict(q=P, k=P, v=P, q_off=P, kv_off=P, kv_len=P, B=1, n_heads=4, n_kv_heads=2, head_dim=64, q_rows=4, kv_rows=9,
             max_q=2, max_kv=9, bf16=False, out=P, workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    pkc.cross_attention(**a)


@pytest.mark.parametrize("kw", [
    dict(q=0), dict(q_off=0), dict(kv_off=0), dict(kv_len=0), dict(out=0), dict(k=0), dict(v=0),
    dict(B=-1), dict(q_rows=-1), dict(kv_rows=-1), dict(max_q=-1), dict(max_kv=-1),
    dict(head_dim=80), dict(head_dim=0), dict(n_heads=0), dict(n_kv_heads=0), dict(n_heads=3), dict(n_kv_heads=-2, n_heads=4),
    dict(q=P + 2), dict(out=P + 8), dict(k=P + 4), dict(v=P + 4), dict(ldq=255), dict(ldq=257), dict(ldk=120), dict(ldv=132),
    dict(ldo=0), dict(ldq=-256), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(q_off=P + 2), dict(kv_off=P + 1), dict(kv_len=P + 3), dict(err=P + 2),
])
def test_cross_attention_refuses(kw):
    refused(cross, **kw)


def test_cross_attention_workspace_is_checked():
    import pkc
    need = pkc.cross_attention_workspace(1, 1, 20000, 4, 2, 64)
    assert need > 0
    big = dict(max_q=1, max_kv=20000, kv_rows=20000)
    assert "workspace" in refused(cross, workspace=0, **big)
    assert "workspace" in refused(cross, workspace_bytes=need - 1, **big)
    assert "workspace" in refused(cross, workspace=P + 4, **big)
    for bad in ((0, 1, 1, 4, 2, 64), (1, 0, 1, 4, 2, 64), (1, 1, -1, 4, 2, 64), (1, 1, 1, 4, 3, 64), (1, 1, 1, 0, 0, 64)):
        assert pkc.cross_attention_workspace(*bad) == 0


CACHES = [dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0), dict(table=0), dict(page=8), dict(page=48), dict(page=256),
          dict(head_dim=96), dict(n_pages=0), dict(n_kv_heads=0), dict(table_ld=0), dict(k=P + 8), dict(v=P + 1)]


@pytest.mark.parametrize("kw", CACHES)
def test_bad_caches_are_refused(kw):
    import pkc
    c = cache(**kw)
    refused(pkc.kv8_append, c, P, P, P, P, 1, rows=1, max_new=1, bf16=True)
    refused(pkc.kv8_attention, c, P, P, P, 1, 4, q_rows=1, max_q=1, max_len=8, bf16=True, out=P)
    refused(pkc.kv8_reorder, c, P, P, 1, 2)
    assert pkc.kv8_attention_workspace(c, 1, 1, 64, 4) == 0


def test_kv8_append_refuses():
    import pkc

    def call(k=P, v=P, off=P, lens=P, n=1, rows=1, max_new=1, **kw):
        pkc.kv8_append(cache(), k, v, off, lens, n, rows=rows, max_new=max_new, bf16=False, **kw)

    for kw in (dict(k=0), dict(v=0), dict(off=0), dict(lens=0), dict(n=-1), dict(rows=-1), dict(max_new=-1), dict(k=P + 2),
               dict(ldk=64), dict(ldv=132), dict(ldk=-128), dict(off=P + 2), dict(lens=P + 1), dict(err=P + 2)):
        refused(call, **kw)
    L = pkc.lib()
    assert L.pkc_kv8_append(None, P, 128, P, 128, P, P, 1, 1, 1, 0, None, None) == pkc.PKC_ERR_ARG
    assert L.pkc_kv8_append(ctypes.byref(cache()), P, 128, P, 128, P, P, 1, 1, 1, 2, None, None) == pkc.PKC_ERR_ARG


def test_kv8_attention_refuses():
    import pkc

    def call(q=P, off=P, lens=P, n=1, heads=4, q_rows=1, max_q=1, max_len=40, out=P, workspace=P, workspace_bytes=1 << 30, **kw):
        pkc.kv8_attention(cache(), q, off, lens, n, heads, q_rows=q_rows, max_q=max_q, max_len=max_len, bf16=False, out=out,
                          workspace=workspace, workspace_bytes=workspace_bytes, **kw)

    for kw in (dict(q=0), dict(off=0), dict(lens=0), dict(out=0), dict(n=-1), dict(heads=0), dict(heads=3), dict(q_rows=-1),
               dict(max_q=-1), dict(max_len=-1), dict(max_len=65), dict(q=P + 2), dict(ldq=130), dict(ldo=64),
               dict(scale=float("nan"))):
        refused(call, **kw)


def test_attention_refuses_what_overflows():
    import pkc
    for scale in (3e38, -3e38):  # times log2(e): an infinity
        assert "scale" in refused(cross, scale=scale)
    assert "2^30" in refused(cross, max_kv=2 ** 30 + 1)
    wide = cache(table_ld=2 ** 27)
    assert "2^30" in refused(pkc.kv8_attention, wide, P, P, P, 1, 4, q_rows=1, max_q=1, max_len=2 ** 30 + 1, bf16=True, out=P)
    assert "scale" in refused(pkc.kv8_attention, wide, P, P, P, 1, 4, q_rows=1, max_q=1, max_len=8, bf16=True, out=P, scale=3e38)


def test_kv8_reorder_refuses():
    import pkc
    for args in ((0, P, 1, 2), (P, 0, 1, 2), (P, P, -1, 2), (P, P, 70000, 2), (P, P, 1, 0), (P, P, 1, 33), (P + 2, P, 1, 2), (P, P + 1, 1, 2)):
        refused(pkc.kv8_reorder, cache(), *args)


def test_beam_select_refuses():
    import pkc

    def call(logits=P, cum=P, finished=0, B=1, K=2, V=10, eos=3, score=P, parent=P, token=P, dtype="f32", **kw):
        pkc.beam_select(logits, cum, finished, B, K, V, eos=eos, score=score, parent=parent, token=token, dtype=dtype, **kw)

    for kw in (dict(logits=0), dict(cum=0), dict(score=0), dict(parent=0), dict(token=0), dict(B=-1), dict(K=0), dict(K=33),
               dict(V=0), dict(eos=-1), dict(eos=10), dict(ld=9), dict(logits=P + 2), dict(logits=P + 1, dtype="f16"),
               dict(cum=P + 2), dict(score=P + 1), dict(parent=P + 2), dict(token=P + 3)):
        refused(call, **kw)
    assert pkc.lib().pkc_beam_select(P, 10, 3, P, None, 1, 2, 10, 0, P, P, P, None, None) == pkc.PKC_ERR_ARG


def test_beam_reorder_refuses():
    import pkc

    def call(state=P, parent=P, B=1, K=2, row_bytes=64, **kw):
        pkc.beam_reorder(state, parent, B, K, row_bytes=row_bytes, **kw)

    for kw in (dict(state=0), dict(parent=0), dict(B=-1), dict(B=70000), dict(K=0), dict(K=33), dict(row_bytes=-1),
               dict(row_stride=63), dict(n_outer=-1), dict(n_outer=70000), dict(n_outer=2, outer_stride=127),
               dict(lens=P, unit_bytes=-1), dict(parent=P + 2), dict(lens=P + 1, unit_bytes=4)):
        refused(call, **kw)


def test_nothing_to_do_is_no_error():
    """Empty calls return at once, whatever the pointers are."""
    import pkc
    cross(B=0, q=0, out=0)
    cross(max_q=0, q=0)
    cross(q_rows=0, q=0)
    pkc.kv8_append(cache(), 0, 0, 0, 0, 0, rows=0, max_new=0, bf16=False)
    pkc.kv8_attention(cache(), 0, 0, 0, 0, 4, q_rows=0, max_q=0, max_len=0, bf16=False, out=0)
    pkc.kv8_reorder(cache(), 0, 0, 0, 2)
    pkc.beam_select(0, 0, 0, 0, 2, 10, eos=0, score=0, parent=0, token=0)
    pkc.beam_reorder(0, 0, 0, 2, row_bytes=64)
    pkc.beam_reorder(0, 0, 2, 2, row_bytes=0)


def test_host_memory_is_refused_or_needs_a_device():
    """Valid sizes with memory that is not the device's: refused, or, without a
    GPU, a CUDA error."""
    import numpy as np
    import pkc
    a = np.zeros(4096, np.float32)
    p = (a.ctypes.data + 15) // 16 * 16
    with pytest.raises(pkc.PkcError) as e:
        pkc.beam_reorder(p, p, 1, 2, row_bytes=64)
    assert e.value.status in (pkc.PKC_ERR_ARG, pkc.PKC_ERR_CUDA)
