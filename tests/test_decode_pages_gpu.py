"""Attention over 8-bit pages whose values lie far apart in size: pages of
zeros, pages begun by a token of zeros, pages 2^60 and more apart. Against the
values that the cache holds, in 64 bits."""
import pytest

from test_decode_gpu import append, make_cache, run_kv8, values

pytestmark = pytest.mark.gpu


def dense(c, s, length):
    """Keys and values [length, Hkv, D] float64 that sequence s's cache holds."""
    import torch
    ids = c["table"][s, : -(-length // c["page"])].long()
    return [(values(c, x)[ids] * c[x + "_scale"][ids].double()[..., None, None]).transpose(1, 2).reshape(
        -1, c["Hkv"], c["D"])[:length] for x in "kv"]


def weights(q, k, scale):
    """Causal softmax weights [H, n, t] of the last n tokens' queries, and the
    bound on the error of a score, as in decode_ref.attention_tolerance."""
    import torch
    n, H, D = q.shape
    t = k.shape[0]
    k = k.repeat_interleave(H // k.shape[1], 1)
    s = torch.einsum("nhd,thd->hnt", q, k) * scale
    S = torch.einsum("nhd,thd->hnt", q.abs(), k.abs()).amax(-1, keepdim=True) * abs(scale)
    sees = t - n + 1 + torch.arange(n, device=q.device)
    s = s.masked_fill(torch.arange(t, device=q.device)[None, None, :] >= sees[None, :, None], float("-inf"))
    return torch.softmax(s, -1), (D + 8) * 2.0 ** -24 * S + 2.0 ** -21


def check(c, s, q, out, length, H, far=None):
    """out [n, H, D] against the cache's contents. A probability is rounded to
    f16: half a step, or, below f16's normal range, 2^-25 and no more than
    itself, of values in units in which the rows kernel keeps a page up to 2^4
    above its own (so 2^-21). far [t]: tokens that may count as zeros."""
    import torch
    k, v = dense(c, s, length)
    n, D = q.shape[0], q.shape[2]
    p, d = weights(q.double(), k, D ** -0.5)
    v = v.repeat_interleave(H // c["Hkv"], 1)
    o = torch.einsum("hnt,thd->nhd", p, v)
    rel = torch.expm1(2 * d) + 2.0 ** -11 + (min(length, 4096) + 8) * 2.0 ** -23
    err = p * rel + p.clamp(max=2.0 ** -21)
    if far is not None:
        err = torch.where(far, err + p, err)
    tol = torch.einsum("hnt,thd->nhd", err, v.abs()) * 1.01 + o.abs() * (torch.finfo(out.dtype).eps / 2) * 1.01
    tol = tol + torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
    got = out.double()
    assert torch.isfinite(got).all()
    bad = ((got - o).abs() - tol).max().item()
    assert bad <= 0, (bad, length)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,length,D", [(150, 420, 64), (150, 420, 128), (140, 1300, 64), (140, 1300, 128), (1, 1300, 64), (20, 420, 128)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_kv8_attention_zero_value_pages(cuda, bf16, n, length, D, page):
    """Pages whose values are all zero for one head (a silent head, padded
    tokens): the first, one inside, several in a row, the last, and a last page
    that one such token has begun. One part of the keys and several; another
    head, whose values are ordinary, beside it."""
    import torch
    dt = torch.bfloat16 if bf16 else torch.float16
    g = torch.Generator().manual_seed(page + length + D)
    H, Hkv = 4, 2
    begun = (length // page) * page + 1
    whole = (length // page) * page
    for zero, t in (([(0, page)], length), ([(page, 2 * page)], length), ([(page, 2 * page), (2 * page, 3 * page)], length),
                    ([(whole - page, whole)], whole), ([(begun - 1, begun)], begun), ([(0, page), (whole - page, length)], length)):
        new = torch.randn(t, 2, Hkv, D, generator=g)
        for lo, hi in zero:
            new[lo:hi, 1, 0] = 0.0
        c = make_cache(cuda, 2, [t, n], Hkv, D, page)
        other = torch.randn(n, 2, Hkv, D, generator=g)
        append(c, torch.cat([new, other]).to(dt).to(cuda), [t, n], [t, n])
        ids = c["table"][0].long()
        assert float(c["v_scale"][ids[zero[-1][0] // page], 0]) == 2.0 ** -126
        q = torch.randn(2 * n, H, D, generator=g).to(dt).to(cuda)
        out = torch.full((2 * n, H * D), -7.0, dtype=dt, device=cuda)
        run_kv8(c, q.view(2 * n, H * D), [n, n], [t, n], H, out)
        assert int(c["err"]) == 0
        out = out.view(2 * n, H, D)
        check(c, 0, q[:n], out[:n], t, H)
        check(c, 1, q[n:], out[n:], n, H)


def scaled_cache(cuda, page, D, exps, g):
    """One sequence of whole pages, one head, random codes, page j's values at
    2^exps[j]; the keys of every second page point where the query does, those
    of the others away from it."""
    import torch
    t = page * len(exps)
    c = make_cache(cuda, 1, [t], 1, D, page)
    for x in "kv":
        c[x].copy_((torch.randn(c[x].shape, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    c["k_scale"].fill_(2.0 ** -7)
    c["v_scale"].fill_(1.0)
    for j, e in enumerate(exps):
        c["v_scale"][int(c["table"][0, j]), 0] = 2.0 ** e
    return c, t


@pytest.mark.parametrize("n", [1, 20, 140])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("low,high", [(-40, 20), (-59, 20), (-12, 8)])
def test_kv8_attention_far_below_with_the_weight(cuda, n, D, page, low, high):
    """Pages of small values between pages of values up to 2^79 larger: where
    the small pages have the weight, their values come out, to their own
    precision."""
    import torch
    g = torch.Generator().manual_seed(page + D + n)
    pages = max(6, 400 // page)
    for pattern in ("after", "before", "between"):
        exps = [low if {"after": j >= pages // 2, "before": j < pages // 2, "between": j % 3 == 1}[pattern] else high for j in range(pages)]
        c, t = scaled_cache(cuda, page, D, exps, g)
        # keys: +u in the pages of small values, -u in the others
        u = torch.randn(D, generator=g).sign()
        for j, e in enumerate(exps):
            k = (u * (1 if e == low else -1)).expand(page, D) * 128 * (1 + torch.rand(page, 1, generator=g) / 4)
            c["k"][int(c["table"][0, j]), 0] = k.to(torch.float8_e4m3fn).view(torch.uint8).to(cuda)
        q = (u * (4.5 if D == 64 else 3.2) + torch.randn(n, 1, D, generator=g) * 0.1).bfloat16().to(cuda)
        out = torch.full((n, D), -7.0, dtype=torch.bfloat16, device=cuda)
        run_kv8(c, q.view(n, D), [n], [t], 1, out)
        assert int(c["err"]) == 0
        got = out.view(n, 1, D)
        check(c, 0, q, got, t, 1)
        # (the test means something: the small pages decide)
        if low > -50 and n == 1:
            assert float(got.abs().max()) < 2.0 ** (low + 10)


@pytest.mark.parametrize("n", [1, 140])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("exps", [[0, -60, 3, -126, -126, 0], [-126, 0, -90, -30], [60, -60, 60, -126], [-126, -100, -50, 0, 50, 90],
                                  [90, 50, 0, -50, -100, -126], [0, -126], [-126, -126], [-7, -126, -7, -126, -7, -126, -7, -126]])
def test_kv8_attention_pages_beyond_all_range(cuda, n, page, exps):
    """Value pages up to 2^216 apart: finite, and right but for pages 2^80
    below the largest, which may count as zeros."""
    import torch
    g = torch.Generator().manual_seed(page + len(exps))
    exps = [e for e in exps for _ in range(2)]
    while len(exps) * page < 140:
        exps = exps + exps
    for D in (64, 128):
        c, t = scaled_cache(cuda, page, D, exps, g)
        q = (torch.randn(n, 1, D, generator=g)).bfloat16().to(cuda)
        out = torch.full((n, D), -7.0, dtype=torch.bfloat16, device=cuda)
        run_kv8(c, q.view(n, D), [n], [t], 1, out)
        far = torch.tensor([e < max(exps) - 80 for e in exps], device=cuda).repeat_interleave(page)
        check(c, 0, q, out.view(n, 1, D), t, 1, far)


@pytest.mark.parametrize("n", [1, 100, 140])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("exps", [[20, -58, 70], [20, -58, 70, -8, 90], [0, -80, 80], [-40, -120, 30, 30, -45, 100], [10, -65, 60, 60, -15]])
def test_kv8_attention_falls_then_rises(cuda, n, page, exps):
    """A page far below the first, then one far above both: a row that sees the
    first keeps its values, which are no more than 2^80 below the largest."""
    import torch
    g = torch.Generator().manual_seed(page + len(exps))
    for rep in (1, max(1, 64 // page), 2 * max(1, 64 // page)):
        each = [e for e in exps for _ in range(rep)]
        if len(each) * page < n:
            continue
        for D in (64, 128):
            c, t = scaled_cache(cuda, page, D, each, g)
            q = (torch.randn(n, 1, D, generator=g) * 0.5).bfloat16().to(cuda)
            out = torch.full((n, D), -7.0, dtype=torch.bfloat16, device=cuda)
            run_kv8(c, q.view(n, D), [n], [t], 1, out)
            far = torch.tensor([e < max(each) - 80 for e in each], device=cuda).repeat_interleave(page)
            check(c, 0, q, out.view(n, 1, D), t, 1, far)
