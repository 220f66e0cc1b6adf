"""The attention decoder's operators at the ends of their types' ranges and
where a call is partly wrong."""
import pytest

from test_decode_gpu import append, make_cache, offsets, run_kv8, run_select, stream, values

pytestmark = pytest.mark.gpu


def test_kv8_attention_tiny_values_long_sums(cuda):
    """Values at the smallest scale (2^-126) under equal weights of 60,000 keys:
    the mean keeps its precision. Codes are multiples of 8 up to 120, so sums
    are whole numbers below 2^24 and exact; what is left is a reciprocal, two
    products and the output's rounding (bf16 keeps 8 bits: half a step is 2^-8
    of the value at most)."""
    import torch
    page, D, H, n, t = 128, 64, 32, 1184, 65000
    c = make_cache(cuda, 1, [t], 1, D, page)
    g = torch.Generator(device=cuda).manual_seed(5)
    code = (torch.randint(8, 16, c["v"].shape, generator=g, device=cuda) * 8).float()
    c["v"].copy_(code.to(torch.float8_e4m3fn).view(torch.uint8))
    c["k"].zero_()
    c["k_scale"].fill_(1.0)
    c["v_scale"].fill_(2.0 ** -126)
    # two sequences of the same pages: as many rows as leave the keys in one part
    c["table"] = c["table"].repeat(2, 1).contiguous()
    c["c"].table = c["table"].data_ptr()
    q = torch.randn(2 * n, H * D, generator=g, device=cuda).bfloat16()
    out = torch.full((2 * n, H * D), -7.0, dtype=torch.bfloat16, device=cuda)
    import pkc
    assert pkc.kv8_attention_workspace(c["c"], 2, n, t, H) == 0
    run_kv8(c, q, [n, n], [t, t], H, out)
    assert int(c["err"]) == 0
    v = code[c["table"][0, : -(-t // page)].long()].double().reshape(-1, D)[:t]
    sees = torch.arange(t - n + 1, t + 1, device=cuda)
    mean = v.cumsum(0)[sees - 1] / sees[:, None] * 2.0 ** -126
    tol = mean * (2.0 ** -8 + 8 * 2.0 ** -24)
    got = out.double().view(2, n, H, D)
    assert ((got - mean[None, :, None]).abs() <= tol[None, :, None]).all()


@pytest.mark.parametrize("n", [1, 20, 140])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("e", [124, -124])
def test_kv8_attention_ordinary_scores_of_extreme_keys(cuda, n, page, e):
    """bf16 keys about 2^124 with queries about 2^-124, and the other way
    round: neither's size alone may leave f32."""
    import decode_ref
    import torch
    g = torch.Generator().manual_seed(page + n)
    t, D = 300, 64
    new = torch.randn(t, 2, 1, D, generator=g)
    new[:, 0] *= 2.0 ** e
    new = new.bfloat16().to(cuda)
    c = make_cache(cuda, 1, [t], 1, D, page)
    append(c, new, [t], [t])
    ids = c["table"][0, : -(-t // page)].long()
    k, v = ((values(c, x)[ids] * c[x + "_scale"][ids].double()[..., None, None]).transpose(1, 2).reshape(-1, 1, D)[:t] for x in "kv")
    q = (torch.randn(n, D, generator=g) * 2.0 ** -e).bfloat16().to(cuda)
    out = torch.full((n, D), -7.0, dtype=torch.bfloat16, device=cuda)
    run_kv8(c, q, [n], [t], 1, out)
    assert int(c["err"]) == 0
    o, A, S = decode_ref.attention(q.double().view(n, 1, D), k, v, D ** -0.5, True)
    tol = decode_ref.attention_tolerance(o, A, S, float(v.abs().max()), t, D, torch.bfloat16, torch.float16)
    got = out.double().view(n, 1, D)
    assert torch.isfinite(got).all() and ((got - o).abs() <= tol).all()


@pytest.mark.parametrize("V", [60, 9000])
def test_beam_select_infinite_scores(cuda, V):
    """A score of +inf offers -inf like one that is not a number, whether its
    row has masked tokens, has finished or neither."""
    import decode_ref
    import torch
    B, K = 4, 4
    g = torch.Generator().manual_seed(V)
    logits = torch.randn(B, K, V, generator=g).to(cuda)
    cum = torch.randn(B, K, generator=g).to(cuda)
    fin = torch.zeros(B, K, dtype=torch.uint8, device=cuda)
    cum[0, 1] = float("inf")
    cum[1, 2] = float("inf")
    logits[1, 2, 3:] = float("-inf")
    cum[2, 0] = float("inf")
    fin[2, 0] = 1
    cum[3] = float("inf")
    score, parent, token, done = run_select(logits, cum, fin, V - 1)
    dead = torch.where(cum == float("inf"), float("-inf"), cum)
    rs, rp, rt, rd = decode_ref.beam_select(logits, dead, fin.bool(), V - 1)
    assert not torch.isnan(score).any()
    assert torch.equal(parent.long(), rp) and torch.equal(token.long(), rt) and torch.equal(done.bool(), rd)
    live = torch.isfinite(rs)
    assert torch.equal(torch.isfinite(score), live) and (score[~live] == float("-inf")).all()
    # exponentials within 2^-22 of their values, so is their sum's logarithm; one rounding to f32
    assert ((score.double() - rs)[live].abs() <= 2.0 ** -21 + rs[live].abs() * 2.0 ** -24 * 1.01).all()


def test_beam_select_close_scores_near_zero(cuda):
    """Hypotheses whose scores are near zero: a score is within 2^-21 of the
    exact one (exponentials within 2^-22 of their values), and two that are
    further apart than twice that come out in their exact order."""
    import decode_ref
    import torch
    B, K, V = 64, 8, 2000
    g = torch.Generator().manual_seed(8)
    row = torch.randn(B, 1, V, generator=g).expand(B, K, V).clone()
    row[:, :, 0] = 30.0
    row[:, :, 1] = 20.0 + torch.rand(B, K, generator=g)
    cum = torch.rand(B, K, generator=g) * 2.0 ** -16
    row, cum = row.to(cuda), cum.to(cuda)
    no = torch.zeros(B, K, dtype=torch.uint8, device=cuda)
    score, parent, token, _ = run_select(row, cum, no, V - 1)
    rs, rp, rt, _ = decode_ref.beam_select(row, cum, no.bool(), V - 1)
    bound = 2.0 ** -21 + rs.abs() * 2.0 ** -24 * 1.01
    assert ((score.double() - rs).abs() <= bound).all()
    # what was picked has, in 64 bits, the score that its place should have, to within the bound of both
    lp = torch.log_softmax(row.double(), -1) + cum.double()[..., None]
    picked = lp.flatten(1).gather(1, parent.long() * V + token.long())
    assert ((picked - rs).abs() <= 2 * 2.0 ** -21).all()


def test_beam_reorder_negative_length_is_reported(cuda):
    """A negative length leaves its item as it is and is reported; the other
    items move. A length of zero is no error."""
    import pkc
    import torch
    for bad in (-1, 0):
        x = torch.arange(12, dtype=torch.float32, device=cuda).view(3, 4, 1).repeat(1, 1, 8).clone()
        before = x.clone()
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        parent = torch.tensor([[3, 2, 1, 0]] * 3, dtype=torch.int32, device=cuda)
        lens = torch.tensor([2, bad, 2], dtype=torch.int32, device=cuda)
        pkc.beam_reorder(x.data_ptr(), parent.data_ptr(), 3, 4, row_bytes=32, lens=lens.data_ptr(), unit_bytes=16,
                         err=err.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        assert int(err) == (110 if bad < 0 else 0)
        assert torch.equal(x[1], before[1])
        for b in (0, 2):
            assert torch.equal(x[b], before[b].flip(0))


@pytest.mark.parametrize("n", [1, 9])
def test_kv8_append_beside_a_bad_sequence(cuda, n):
    """A sequence that is left out (a bad page, length or offset) changes
    nothing of the other one's: its codes and scales are those of a call of its
    own."""
    import torch
    new = torch.randn(2 * n, 2, 1, 64, generator=torch.Generator().manual_seed(2)).half().to(cuda)
    alone = make_cache(cuda, 2, [n, n], 1, 64, 16)
    append(alone, new[:n].contiguous(), [n, 0], [n, 0], max_new=n)
    assert int(alone["err"]) == 0
    for what in ("page", "negative page", "length", "short length", "offset"):
        c = make_cache(cuda, 2, [n, n], 1, 64, 16)
        mine = int(c["table"][0, 0])
        lens, n_new = [n, n], [n, n]
        if what == "page":
            c["table"][1] = c["total"]
        elif what == "negative page":
            c["table"][1] = -5
        elif what == "length":
            lens = [n, 16 * c["table"].shape[1] + 1]
        elif what == "short length":
            lens = [n, n - 1]
        else:
            n_new = [n, n + 3]
        append(c, new, n_new, lens, max_new=n)
        assert int(c["err"]) == 110, what
        for x in "kv":
            assert torch.equal(c[x][mine], alone[x][mine]), what
            assert torch.equal(c[x + "_scale"][mine], alone[x + "_scale"][mine]), what
            others = [p for p in range(c["total"]) if p != mine]
            assert (c[x][others] == 0x7f).all(), what
        live = values(c, "k")[mine, 0, :n]
        assert torch.isfinite(live).all() and (live != 0).any()


def test_cross_attention_bound_beyond_a_grid_is_refused(cuda):
    """A max_q so loose that its tiles pass a grid's size: an error, not a
    wrapped number of tiles that leaves rows out. The largest that fits is
    answered in full."""
    import pkc
    import torch
    H, D, n = 512, 64, 2
    q = torch.randn(n, H * D, device=cuda).half()
    kv = torch.randn(9, 2, D, device=cuda).half()
    out = torch.full_like(q, -7.0)
    off, zero, nine = offsets([n], cuda), torch.zeros(1, dtype=torch.int32, device=cuda), torch.full((1,), 9, dtype=torch.int32, device=cuda)

    def call(max_q):
        pkc.cross_attention(q.data_ptr(), kv.data_ptr(), kv[:, 1].data_ptr(), off.data_ptr(), zero.data_ptr(), nine.data_ptr(), 1,
                            H, 1, D, q_rows=n, kv_rows=9, max_q=max_q, max_kv=9, bf16=False, out=out.data_ptr(), ldk=2 * D,
                            ldv=2 * D, stream=stream())
        torch.cuda.synchronize()

    with pytest.raises(pkc.PkcError):
        call((1 << 30) + 1)  # 2^32 + 4 tiles of 128 rows
    assert (out == -7).all()
    call(2000)
    s = torch.einsum("nhd,td->nht", q.double().view(n, H, D), kv[:, 0].double()) * D ** -0.5
    ref = torch.einsum("nht,td->nhd", torch.softmax(s, -1), kv[:, 1].double()).flatten(1)
    # weights and output are rounded to f16, half a step each
    assert ((out.double() - ref).abs() <= float(kv.abs().max()) * 2.0 ** -10 + 2.0 ** -20).all()


@pytest.mark.parametrize("bound", [(1 << 31) - 1, (1 << 31) - 15, 1 << 20])
def test_kv8_append_loosest_bounds(cuda, bound):
    """rows and max_new as loose as an int allows: every sequence is written as
    with the true bounds."""
    import pkc
    import torch
    Hkv, D, lens = 128, 64, [20, 33]
    g = torch.Generator().manual_seed(1)
    new = torch.randn(sum(lens), 2, Hkv, D, generator=g).half().to(cuda)
    want, got = (make_cache(cuda, 2, lens, Hkv, D, 16) for _ in range(2))
    append(want, new, lens, lens)
    off, ln = offsets(lens, cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    pkc.kv8_append(got["c"], new.data_ptr(), new[:, 1].data_ptr(), off.data_ptr(), ln.data_ptr(), 2, rows=bound, max_new=bound,
                   ldk=new.stride(0), ldv=new.stride(0), bf16=False, err=got["err"].data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert int(got["err"]) == 0
    for x in "kv":
        assert torch.equal(got[x], want[x])
        assert torch.equal(got[x + "_scale"].nan_to_num(-1.0), want[x + "_scale"].nan_to_num(-1.0))
