"""The attention decoder's operators (cross attention, 8-bit cache, beam
selection, reordering) through the C ABI against 64-bit restatements
(decode_ref.py, which also derives the bounds)."""
import math

import pytest

pytestmark = pytest.mark.gpu


def offsets(lens, dev):
    import torch
    t = torch.zeros(len(lens) + 1, dtype=torch.int32)
    t[1:] = torch.tensor(lens, dtype=torch.int32).cumsum(0)
    return t.to(dev)


def workspace(n, dev):
    import torch
    return torch.full((max(16, n),), 0xff, dtype=torch.uint8, device=dev)


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------- cross attention


def run_cross(cuda, q, kv, q_lens, kv_off, kv_lens, H, Hkv, D, out, *, scale=None, max_q=None, max_kv=None, err=None,
              q_off=None):
    """q / out [rows, ld], kv [rows, 2, Hkv, D + pad] (their strides are passed on)."""
    import pkc
    import torch
    B = len(kv_lens)
    max_q = max(q_lens) if max_q is None else max_q
    max_kv = max(kv_lens) if max_kv is None else max_kv
    ws = workspace(pkc.cross_attention_workspace(B, max_q, max_kv, H, Hkv, D), cuda)
    qo = offsets(q_lens, cuda) if q_off is None else q_off
    ko = torch.tensor(kv_off, dtype=torch.int32, device=cuda)
    kl = torch.tensor(kv_lens, dtype=torch.int32, device=cuda)
    pkc.cross_attention(q.data_ptr(), kv.data_ptr(), kv[:, 1].data_ptr(), qo.data_ptr(), ko.data_ptr(), kl.data_ptr(),
                        B, H, Hkv, D, q_rows=q.shape[0], kv_rows=kv.shape[0], max_q=max_q, max_kv=max_kv,
                        ldq=q.stride(0), ldk=kv.stride(0), ldv=kv.stride(0), ldo=out.stride(0), scale=scale,
                        bf16=q.dtype == torch.bfloat16, out=out.data_ptr(), workspace=ws.data_ptr(),
                        workspace_bytes=ws.numel(), err=0 if err is None else err.data_ptr(), stream=stream())
    torch.cuda.synchronize()


def check_cross(cuda, q_lens, kv_lens, H, Hkv, D, bf16, *, seed=0, gap=3, q_scale=1.0, scale=None, max_q=None):
    """Items apart from one another by `gap` rows of NaN, strided rows, and
    rows of q and out behind the last item."""
    import decode_ref
    import torch
    dt = torch.bfloat16 if bf16 else torch.float16
    g = torch.Generator().manual_seed(seed + sum(q_lens) * 7 + sum(kv_lens))
    M = sum(q_lens)
    q = torch.full((M + 2, H * D + 16), float("nan"), dtype=dt)
    q[:M, :H * D] = (torch.randn(M, H * D, generator=g) * q_scale).to(dt)
    q[M:] = 1.0
    kv_off, at = [], gap
    for t in kv_lens:
        kv_off.append(at)
        at += t + gap
    kv = torch.full((at, 2, Hkv * D + 8), float("nan"), dtype=dt)
    for o, t in zip(kv_off, kv_lens):
        kv[o:o + t, :, :Hkv * D] = torch.randn(t, 2, Hkv * D, generator=g).to(dt)
    q, kv = q.to(cuda), kv.to(cuda)
    out = torch.full((M + 2, H * D + 8), -7.0, dtype=dt, device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    run_cross(cuda, q, kv, q_lens, kv_off, kv_lens, H, Hkv, D, out, err=err, scale=scale, max_q=max_q)
    assert int(err) == 0
    assert (out[M:] == -7).all() and (out[:, H * D:] == -7).all()
    r0 = 0
    for n, o, t in zip(q_lens, kv_off, kv_lens):
        qi = q[r0:r0 + n, :H * D].double().view(n, H, D)
        k, v = (kv[o:o + t, x, :Hkv * D].double().view(t, Hkv, D) for x in (0, 1))
        sc = D ** -0.5 if scale is None else scale
        ref, A, S = decode_ref.attention(qi, k, v, sc, False)
        tol = decode_ref.attention_tolerance(ref, A, S, float(v.abs().max()) if t else 0.0, t, D, dt, dt)
        got = out[r0:r0 + n, :H * D].double().view(n, H, D)
        assert torch.isfinite(got).all()
        bad = ((got - ref).abs() - tol).max().item() if n else -1
        assert bad <= 0, (bad, n, t)
        r0 += n


CROSS = [
    # (query rows, keys, H, Hkv, D)
    ([1], [1], 1, 1, 64),
    ([1], [437], 8, 8, 128),
    ([1, 0, 2, 1], [5, 9, 0, 17], 4, 4, 64),
    ([8, 8, 8], [25, 437, 131], 8, 8, 128),
    ([5, 3, 16, 17], [16, 15, 33, 64], 8, 2, 64),
    ([1, 1], [5000, 129], 8, 1, 128),
    ([33, 1, 70], [300, 63, 1], 4, 2, 128),
    ([200, 130, 7], [437, 128, 513], 4, 4, 128),
    ([129, 257], [64, 191], 8, 2, 64),
    ([300], [1500], 6, 3, 64),
    # heads that share a key head in odd numbers, and many of them
    ([1, 2], [70, 33], 3, 1, 128),
    ([60, 7], [100, 65], 6, 2, 64),
    ([40, 1, 30], [129, 20, 64], 5, 1, 128),
    ([1, 3], [300, 50], 24, 1, 64),
    ([9, 20], [77, 210], 24, 1, 128),
]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("q_lens,kv_lens,H,Hkv,D", CROSS)
def test_cross_attention(cuda, bf16, q_lens, kv_lens, H, Hkv, D):
    check_cross(cuda, q_lens, kv_lens, H, Hkv, D, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("q_lens,kv_lens,H,Hkv,D", [
    ([36], [500], 8, 8, 64), ([64, 0, 50], [200, 9, 0], 4, 4, 128), ([12, 11, 9] * 14, [7, 130, 64] * 14, 4, 1, 64),
    ([16, 15], [390, 17], 4, 1, 128), ([150], [3001], 2, 1, 128), ([9, 70, 1], [2500, 300, 1100], 3, 3, 64),
])
def test_cross_attention_between_few_and_many_rows(cuda, bf16, q_lens, kv_lens, H, Hkv, D):
    """33 to 64 rows (blocks of 16, or a tile), and parts of one item's keys."""
    check_cross(cuda, q_lens, kv_lens, H, Hkv, D, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [1, 200])
def test_cross_attention_long_and_peaked(cuda, bf16, n):
    """Many keys, and scores so far apart that one key has nearly all weight."""
    check_cross(cuda, [n], [20011], 2, 1, 64, bf16)
    check_cross(cuda, [n, 3], [700, 90], 4, 2, 128, bf16, q_scale=20.0)


@pytest.mark.parametrize("D", [64, 128])
def test_cross_attention_many_rows_without_keys(cuda, D):
    """Tiles of rows that have no key give zeros, all of them."""
    for seed in range(3):
        check_cross(cuda, [88, 68, 14, 112, 76, 25, 128, 130, 70] * 9, [2, 0, 0, 0, 2, 0, 0, 0, 0] * 9, 4, 4, D, False,
                    seed=seed)


@pytest.mark.parametrize("n", [2, 150])
def test_cross_attention_max_q_above_the_rows(cuda, n):
    """max_q is a bound: a larger one changes nothing."""
    check_cross(cuda, [n, 1], [100, 77], 4, 4, 64, False, max_q=400)


@pytest.mark.parametrize("n", [3, 140])
def test_cross_attention_extreme_scores(cuda, n):
    """All scores equal and hugely negative (a mask of the type's lowest value
    added upstream): weights stay even, nothing is NaN."""
    import torch
    D, t = 64, 90
    q = torch.full((n, D), -240.0, dtype=torch.float16, device=cuda)
    kv = torch.full((t, 2, 1, D), 250.0, dtype=torch.float16, device=cuda)
    kv[:, 1] = torch.arange(t, device=cuda).half()[:, None, None]
    out = torch.zeros(n, D, dtype=torch.float16, device=cuda)
    run_cross(cuda, q, kv, [n], [0], [t], 1, 1, D, out, scale=100.0)
    # weights 1/90 rounded once (2^-11), output once (2^-11), f32 sums
    assert ((out.double() - (t - 1) / 2).abs() <= (t - 1) / 2 * 2.2 * 2.0 ** -11).all()


@pytest.mark.parametrize("n", [3, 140])
def test_cross_attention_nan_stays_in_its_item(cuda, n):
    """A NaN or an infinity in one item's keys or values is that item's alone."""
    import torch
    D, t = 64, 70
    g = torch.Generator().manual_seed(5)
    q = torch.randn(3 * n, 2 * D, generator=g).half().to(cuda)
    kv = torch.randn(3 * t, 2, 2, D, generator=g).half().to(cuda)
    want = torch.zeros(3 * n, 2 * D, dtype=torch.float16, device=cuda)
    run_cross(cuda, q, kv, [n] * 3, [0, t, 2 * t], [t] * 3, 2, 2, D, want)
    kv[t + 3, 0, 0, 1] = float("nan")
    kv[2 * t - 1, 1, 1, 5] = float("inf")
    out = torch.zeros_like(want)
    run_cross(cuda, q, kv, [n] * 3, [0, t, 2 * t], [t] * 3, 2, 2, D, out)
    assert torch.equal(out[:n], want[:n]) and torch.equal(out[2 * n:], want[2 * n:])
    assert torch.isnan(out[n:2 * n, :D]).all()
    assert torch.isinf(out[n:2 * n, D + 5]).all()
    keep = [c for c in range(D, 2 * D) if c != D + 5]
    assert torch.equal(out[n:2 * n][:, keep], want[n:2 * n][:, keep])


@pytest.mark.parametrize("n", [3, 140])
def test_cross_attention_without_any_keys(cuda, n):
    """kv_rows = 0 and no key memory at all: zeros."""
    import pkc
    import torch
    q = torch.randn(n, 128, generator=torch.Generator().manual_seed(1)).half().to(cuda)
    out = torch.full_like(q, -7.0)
    z = torch.zeros(2, dtype=torch.int32, device=cuda)
    qo = offsets([n - 1, 1], cuda)
    pkc.cross_attention(q.data_ptr(), 0, 0, qo.data_ptr(), z.data_ptr(), z.data_ptr(), 2, 2, 2, 64, q_rows=n, kv_rows=0,
                        max_q=n, max_kv=0, bf16=False, out=out.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert (out == 0).all()


@pytest.mark.parametrize("n", [2, 150])
def test_cross_attention_beyond_32_bits(cuda, n):
    """Keys whose rows lie behind the 2^32nd byte of their memory."""
    import torch
    D, t, ld = 64, 90, 65536
    rows = (1 << 32) // (2 * ld) + t + 10
    big = torch.empty(rows, ld, dtype=torch.float16, device=cuda)
    g = torch.Generator().manual_seed(14)
    kv = torch.randn(t, 2, 1, D, generator=g).half().to(cuda)
    big[-t:, :2 * D] = kv.view(t, 2 * D)
    q = torch.randn(n, D, generator=g).half().to(cuda)
    want, out = torch.zeros_like(q), torch.zeros_like(q)
    run_cross(cuda, q, kv, [n], [0], [t], 1, 1, D, want)
    run_cross(cuda, q, big.as_strided((rows, 2, 1, D), (ld, D, D, 1)), [n], [rows - t], [t], 1, 1, D, out)
    assert torch.equal(out, want) and float(out.abs().max()) > 0


@pytest.mark.parametrize("n", [4, 140])
def test_cross_attention_bad_tables_are_reported(cuda, n):
    """Offsets and lengths beyond the sizes of the call: that item is left
    out, the others are served, the error word says so."""
    import torch
    D, t = 64, 40
    g = torch.Generator().manual_seed(6)
    q = torch.randn(2 * n, D, generator=g).half().to(cuda)
    kv = torch.randn(2 * t, 2, 1, D, generator=g).half().to(cuda)
    want = torch.zeros(2 * n, D, dtype=torch.float16, device=cuda)
    run_cross(cuda, q, kv, [n, n], [0, t], [t, t], 1, 1, D, want)
    for off, lens, qo in (([0, t + 1], [t, t], None), ([0, -1], [t, t], None), ([0, t], [t, t + 1], None),
                          ([0, t], [t, -1], None), ([0, t], [t, t], [0, n, n - 1]), ([0, t], [t, t], [0, n, 2 * n + 1])):
        out = torch.full_like(want, -7.0)
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        qo = None if qo is None else torch.tensor(qo, dtype=torch.int32, device=cuda)
        run_cross(cuda, q, kv, [n, n], off, lens, 1, 1, D, out, err=err, max_kv=t, q_off=qo)
        assert int(err) == 110
        assert torch.equal(out[:n], want[:n]) and (out[n:] == -7).all()


# ---------------------------------------------------------------- the 8-bit cache


def make_cache(cuda, S, lens, Hkv, D, page, *, seed=0, fill=0x7f, spare=2):
    """Device pools full of NaN codes and a table of shuffled pages."""
    import pkc
    import torch
    need = [-(-n // page) for n in lens]
    width, total = max(1, max(need)) + 1, sum(need) + spare
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((S, width), -1, dtype=torch.int32)
    for s in range(S):
        for p in range(need[s]):
            table[s, p] = perm.pop()
    c = {"table": table.to(cuda), "page": page, "Hkv": Hkv, "D": D, "total": total}
    for x in "kv":
        c[x] = torch.full((total, Hkv, page, D), fill, dtype=torch.uint8, device=cuda)
        c[x + "_scale"] = torch.full((total, Hkv), float("nan"), device=cuda)
    c["c"] = pkc.KV8Cache(k=c["k"].data_ptr(), v=c["v"].data_ptr(), k_scale=c["k_scale"].data_ptr(),
                          v_scale=c["v_scale"].data_ptr(), table=c["table"].data_ptr(), n_pages=total, page=page,
                          n_kv_heads=Hkv, head_dim=D, table_ld=width)
    c["err"] = torch.zeros(1, dtype=torch.int32, device=cuda)
    return c


def append(c, new, n_new, lens, *, max_new=None):
    """new [rows, 2, Hkv, D + pad] 16-bit."""
    import pkc
    import torch
    dev = new.device
    no, ln = offsets(n_new, dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    pkc.kv8_append(c["c"], new.data_ptr(), new[:, 1].data_ptr(), no.data_ptr(), ln.data_ptr(), len(lens),
                   rows=new.shape[0], max_new=max(n_new) if max_new is None else max_new, ldk=new.stride(0),
                   ldv=new.stride(0), bf16=new.dtype == torch.bfloat16, err=c["err"].data_ptr(), stream=stream())
    torch.cuda.synchronize()


def values(c, x):
    import torch
    return c[x].view(torch.float8_e4m3fn).double()


def check_pools(c, ref, touched_slots):
    """Codes and scales equal the restatement's where tokens lie; elsewhere the
    bytes are what they were."""
    import torch
    for i, x in enumerate("kv"):
        got, sc = values(c, x).cpu(), c[x + "_scale"].cpu()
        m = touched_slots[:, None, :, None].expand_as(got)
        assert torch.equal(got[m], ref.code[i][m])
        assert (c[x].cpu()[~m] == 0x7f).all()
        used = touched_slots.any(-1)
        assert torch.equal(sc[used].double(), torch.exp2(ref.exp[i][used].double()))
        assert torch.isnan(sc[~used]).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("Hkv,D,page", [(2, 64, 16), (1, 128, 32), (3, 64, 64), (2, 128, 128)])
def test_kv8_append(cuda, bf16, Hkv, D, page):
    """Several appends of uneven lengths (none, one, many; across page ends),
    values of growing and shrinking size: codes and scales bit for bit."""
    import decode_ref
    import torch
    dt = torch.bfloat16 if bf16 else torch.float16
    steps = [[0, 3, page, 2 * page + 5], [1, 1, 1, 1], [1, 0, page - 1, 7], [page + 1, 2, 0, 1], [1, 1, 1, 1]]
    S = 4
    total = [sum(s[i] for s in steps) for i in range(S)]
    c = make_cache(cuda, S, total, Hkv, D, page)
    ref = decode_ref.RefCache(c["total"], Hkv, page, D)
    slots = torch.zeros(c["total"], page, dtype=torch.bool)
    g = torch.Generator().manual_seed(page + D)
    lens = [0] * S
    for step, n_new in enumerate(steps):
        rows = sum(n_new)
        new = torch.full((rows + 1, 2, Hkv, D + 8), float("nan"), dtype=dt)
        size = torch.exp2(torch.randint(-6, 7, (rows, 2, Hkv, 1), generator=g).float())
        new[:rows, ..., :D] = (torch.randn(rows, 2, Hkv, D, generator=g) * size).to(dt)
        if step == 1:
            new[0, 0, 0, :D] = 0.0
        # packed heads: the kernel reads [row][Hkv][D]
        packed = torch.cat([new[..., :D].reshape(rows + 1, 2, Hkv * D), torch.full((rows + 1, 2, 8), float("nan"), dtype=dt)], -1)
        lens = [a + b for a, b in zip(lens, n_new)]
        append(c, packed.to(cuda), n_new, lens)
        r0 = 0
        for s in range(S):
            ref.append(c["table"][s].tolist(), packed[r0:r0 + n_new[s], :, :Hkv * D].double().view(-1, 2, Hkv, D), lens[s])
            for t in range(lens[s] - n_new[s], lens[s]):
                slots[int(c["table"][s, t // page]), t % page] = True
            r0 += n_new[s]
        assert int(c["err"]) == 0
        check_pools(c, ref, slots)


@pytest.mark.parametrize("n", [1, 40])
def test_kv8_append_twice_is_once(cuda, n):
    """The same append again (a replayed graph whose lengths did not move)
    leaves the same bytes."""
    import torch
    c = make_cache(cuda, 2, [70, 60], 2, 64, 32)
    g = torch.Generator().manual_seed(1)
    old = (torch.randn(40, 2, 2, 64, generator=g)).half().to(cuda)
    append(c, old, [20, 20], [20, 20])
    new = (torch.randn(2 * n, 2, 2, 64, generator=g) * 9).half().to(cuda)
    append(c, new, [n, n], [20 + n, 20 + n])
    a = [c[x].clone() for x in ("k", "v", "k_scale", "v_scale")]
    append(c, new, [n, n], [20 + n, 20 + n])
    for x, y in zip(("k", "v", "k_scale", "v_scale"), a):
        assert torch.equal(c[x].view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("n", [1, 40])
def test_kv8_append_loose_bound(cuda, n):
    """max_new far above what comes writes the same bytes."""
    import torch
    g = torch.Generator().manual_seed(2)
    new = torch.randn(2 * n, 2, 2, 64, generator=g).half().to(cuda)
    got = []
    for bound in (n, 2 ** 31 - 1):
        c = make_cache(cuda, 2, [n, n], 2, 64, 16)
        append(c, new, [n, n], [n, n], max_new=bound)
        assert int(c["err"]) == 0
        got.append([c[x].view(torch.uint8).clone() for x in ("k", "v", "k_scale", "v_scale")])
    for x, y in zip(*got):
        assert torch.equal(x, y)


@pytest.mark.parametrize("n", [2, 20])
def test_kv8_append_special_values(cuda, n):
    """Infinities take the largest code and set no scale, a NaN is stored as 0
    and reported, zeros and the smallest values keep the smallest scale."""
    import torch
    c = make_cache(cuda, 1, [n], 1, 64, 32)
    new = torch.zeros(n, 2, 1, 64, dtype=torch.bfloat16)
    new[0, 0, 0, :4] = torch.tensor([float("inf"), float("-inf"), 1.0, float("nan")])
    new[1, 0, 0, 0] = 448.0
    append(c, new.to(cuda), [n], [n])
    p = int(c["table"][0, 0])
    k = values(c, "k")[p, 0]
    assert float(c["k_scale"][p, 0]) == 1.0 and float(c["v_scale"][p, 0]) == 2.0 ** -126
    assert k[0, :4].tolist() == [448.0, -448.0, 1.0, 0.0] and float(k[1, 0]) == 448.0
    assert (values(c, "v")[p, 0, :n] == 0).all()
    assert int(c["err"]) == 111
    big = torch.full((n, 2, 1, 64), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16, device=cuda)
    c["err"].zero_()
    append(c, big, [n], [n])
    assert float(c["k_scale"][p, 0]) == 2.0 ** 120 and int(c["err"]) == 0
    assert (values(c, "k")[p, 0, :n] * 2.0 ** 120 == to_nearest(torch.finfo(torch.bfloat16).max)).all()


def to_nearest(x):
    """x rounded to 4 significant bits."""
    e = 2.0 ** (math.floor(math.log2(x)) - 3)
    return round(x / e) * e


@pytest.mark.parametrize("n", [1, 9])
def test_kv8_append_bad_tables_are_reported(cuda, n):
    """A page, length or offset outside the sizes of the call leaves that
    sequence out and is reported; the other sequence is written."""
    import torch
    for what in ("page", "negative page", "length", "short length", "offset"):
        c = make_cache(cuda, 2, [n, n], 1, 64, 16)
        new = torch.randn(2 * n, 2, 1, 64, generator=torch.Generator().manual_seed(2)).half().to(cuda)
        lens, n_new, max_new = [n, n], [n, n], n
        keep = c["table"].clone()
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
        append(c, new, n_new, lens, max_new=max_new)
        assert int(c["err"]) == 110, what
        assert (c["k"][keep[1, 0].item()] == 0x7f).all()
        assert (values(c, "k")[keep[0, 0].item(), 0, :n] == values(c, "k")[keep[0, 0].item(), 0, :n]).all()


def run_kv8(c, q, q_lens, lens, H, out, *, max_q=None, max_len=None, scale=None):
    import pkc
    import torch
    dev = q.device
    max_q = max(q_lens) if max_q is None else max_q
    max_len = max(lens) if max_len is None else max_len
    ws = workspace(pkc.kv8_attention_workspace(c["c"], len(lens), max_q, max_len, H), dev)
    qo, ln = offsets(q_lens, dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    pkc.kv8_attention(c["c"], q.data_ptr(), qo.data_ptr(), ln.data_ptr(), len(lens), H, q_rows=q.shape[0], max_q=max_q,
                      max_len=max_len, bf16=q.dtype == torch.bfloat16, out=out.data_ptr(), ldq=q.stride(0),
                      ldo=out.stride(0), scale=scale, workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                      err=c["err"].data_ptr(), stream=stream())
    torch.cuda.synchronize()


def check_kv8(cuda, q_lens, lens, H, Hkv, D, page, bf16, *, spread=0, q_scale=1.0):
    """Caches filled by random codes and scales (2^+-spread apart); NaN codes
    behind each sequence's last token."""
    import decode_ref
    import torch
    dt = torch.bfloat16 if bf16 else torch.float16
    S = len(lens)
    c = make_cache(cuda, S, lens, Hkv, D, page)
    ref = decode_ref.RefCache(c["total"], Hkv, page, D)
    g = torch.Generator().manual_seed(sum(lens) + page + D + H)
    ref.code = decode_ref.to_e4m3(torch.randn(2, c["total"], Hkv, page, D, generator=g, dtype=torch.float64) * 100)
    ref.exp = torch.randint(-7 - spread, -6 + spread, (2, c["total"], Hkv), generator=g)
    if spread:  # keys keep scores in a range, values may differ by far
        ref.exp[0] = torch.randint(-9, -6, (c["total"], Hkv), generator=g)
    table = c["table"].tolist()
    live = torch.zeros(c["total"], page, dtype=torch.bool)
    for s in range(S):
        for t in range(lens[s]):
            live[table[s][t // page], t % page] = True
    for i, x in enumerate("kv"):
        codes = ref.code[i].float().to(torch.float8_e4m3fn).view(torch.uint8)
        c[x].copy_(torch.where(live[:, None, :, None], codes, torch.full_like(codes, 0x7f)))
        c[x + "_scale"].copy_(torch.exp2(ref.exp[i].float()))
    M = sum(q_lens)
    q = torch.full((M + 1, H * D + 8), float("nan"), dtype=dt)
    q[:M, :H * D] = (torch.randn(M, H * D, generator=g) * q_scale).to(dt)
    q = q.to(cuda)
    out = torch.full((M + 1, H * D + 8), -7.0, dtype=dt, device=cuda)
    run_kv8(c, q, q_lens, lens, H, out)
    assert int(c["err"]) == 0
    assert (out[M:] == -7).all() and (out[:, H * D:] == -7).all()
    r0 = 0
    for s, (n, t) in enumerate(zip(q_lens, lens)):
        k, v = (y.to(cuda) for y in ref.dense(table[s], t))
        qi = q[r0:r0 + n, :H * D].double().view(n, H, D)
        o, A, S_ = decode_ref.attention(qi, k, v, D ** -0.5, True)
        # probabilities are f16 whatever the queries' type
        tol = decode_ref.attention_tolerance(o, A, S_, 0.0, t, D, dt, torch.float16)
        # below f16's normal range: 2^-25 of each page's own values
        tol = tol + 1.01 * 2.0 ** -25 * v.abs().sum(0).repeat_interleave(H // Hkv, 0)[None] if t else tol
        got = out[r0:r0 + n, :H * D].double().view(n, H, D)
        assert torch.isfinite(got).all()
        bad = ((got - o).abs() - tol).max().item() if n else -1
        assert bad <= 0, (bad, s, n, t)
        r0 += n


KV8 = [
    # (new rows, lengths, H, Hkv, D, page)
    ([1], [1], 1, 1, 64, 16),
    ([1, 0, 1, 1], [17, 4, 16, 129], 4, 4, 64, 16),
    ([1, 1, 1], [448, 31, 33], 8, 8, 128, 32),
    ([1, 1], [3000, 65], 16, 2, 128, 64),
    ([1, 1], [1000, 130], 4, 1, 64, 128),
    ([2, 5, 17], [2, 100, 17], 8, 2, 64, 32),
    ([40, 3, 64], [200, 64, 64], 4, 2, 128, 16),
    ([130, 9, 257], [130, 500, 700], 4, 4, 64, 64),
    ([200, 129], [513, 129], 8, 2, 128, 128),
    ([140, 33], [400, 47], 4, 1, 128, 32),
    ([1, 3], [90, 40], 12, 1, 128, 16),
    ([50, 11], [95, 60], 7, 1, 64, 32),
    ([70], [333], 6, 2, 128, 128),
]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("q_lens,lens,H,Hkv,D,page", KV8)
def test_kv8_attention(cuda, bf16, q_lens, lens, H, Hkv, D, page):
    check_kv8(cuda, q_lens, lens, H, Hkv, D, page, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("q_lens,lens,H,Hkv,D,page", [
    ([16], [500], 16, 4, 128, 64), ([16, 5, 1], [333, 70, 1], 8, 2, 64, 16), ([12, 9] * 35, [163, 40] * 35, 16, 4, 64, 32),
    ([9, 12, 8], [1500, 2048, 700], 16, 4, 128, 128), ([12, 3], [3000, 999], 16, 4, 128, 32), ([256], [5000], 4, 1, 64, 64),
    ([16, 2], [2500, 129], 16, 4, 64, 16),
])
def test_kv8_attention_between_few_and_many_rows(cuda, bf16, q_lens, lens, H, Hkv, D, page):
    """33 to 64 rows (blocks of 16, or a tile), and parts of one sequence's tokens."""
    check_kv8(cuda, q_lens, lens, H, Hkv, D, page, bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [1, 150])
@pytest.mark.parametrize("page", [16, 64])
def test_kv8_attention_pages_far_apart(cuda, bf16, n, page):
    """Value scales of pages up to 2^24 apart, and peaked scores: the page
    that has the weight counts, however small its values are."""
    check_kv8(cuda, [n, n], [700, n], 4, 2, 64, page, bf16, spread=12)
    check_kv8(cuda, [n], [500], 2, 1, 128, page, bf16, spread=12, q_scale=12.0)


@pytest.mark.parametrize("n", [1, 140])
def test_kv8_attention_large_queries(cuda, n):
    """bf16 queries beyond f16's range (2^20) with keys small enough that the
    scores stay ordinary."""
    import decode_ref
    import torch
    c = make_cache(cuda, 1, [200], 1, 64, 32)
    g = torch.Generator().manual_seed(9)
    new = torch.randn(200, 2, 1, 64, generator=g)
    new[:, 0] *= 2.0 ** -22
    new = new.bfloat16().to(cuda)
    append(c, new, [200], [200])
    ref = decode_ref.RefCache(c["total"], 1, 32, 64)
    ref.append(c["table"][0].tolist(), new.double().cpu(), 200)
    k, v = (y.to(cuda) for y in ref.dense(c["table"][0].tolist(), 200))
    q = (torch.randn(n, 64, generator=g) * 2.0 ** 21).bfloat16().to(cuda)
    out = torch.zeros(n, 64, dtype=torch.bfloat16, device=cuda)
    run_kv8(c, q, [n], [200], 1, out)
    o, A, S = decode_ref.attention(q.double().view(n, 1, 64), k, v, 0.125, True)
    tol = decode_ref.attention_tolerance(o, A, S, float(v.abs().max()), 200, 64, torch.bfloat16, torch.float16)
    assert ((out.double().view(n, 1, 64) - o).abs() <= tol).all()


@pytest.mark.parametrize("n", [1, 140])
def test_kv8_attention_bad_tables_are_reported(cuda, n):
    """A page that is none: its tokens are left out; a length beyond max_len
    or below the new rows: the sequence is left out. Both are reported."""
    import torch
    c = make_cache(cuda, 2, [160, 160], 1, 64, 16, fill=0x38)  # code of 1.0
    for x in "kv":
        c[x + "_scale"].fill_(1.0)
    q = torch.randn(2 * n, 64, generator=torch.Generator().manual_seed(3)).half().to(cuda)
    out = torch.full((2 * n, 64), -7.0, dtype=torch.float16, device=cuda)
    for bad in (c["total"], -1):
        keep = int(c["table"][1, 4])
        c["table"][1, 4] = bad
        c["err"].zero_()
        run_kv8(c, q, [n, n], [160, 160], 1, out)
        c["table"][1, 4] = keep
        assert int(c["err"]) == 110
        assert (out == 1.0).all()  # every value that is seen is 1
    for lens in ([160, 161], [160, n - 1]):
        out.fill_(-7.0)
        c["err"].zero_()
        run_kv8(c, q, [n, n], lens, 1, out, max_len=160)
        assert int(c["err"]) == 110
        assert (out[:n] == 1.0).all() and (out[n:] == -7).all()


def test_kv8_pool_beyond_32_bits(cuda):
    """Pages behind the 2^32nd byte of a pool."""
    import pkc
    import torch
    page, Hkv, D = 128, 8, 128
    total = (1 << 32) // (page * Hkv * D) + 3
    pools = {x: torch.empty(total, Hkv, page, D, dtype=torch.uint8, device=cuda) for x in "kv"}
    scales = {x: torch.ones(total, Hkv, device=cuda) for x in "kv"}
    table = torch.tensor([[total - 1, total - 2]], dtype=torch.int32, device=cuda)
    c = {"c": pkc.KV8Cache(k=pools["k"].data_ptr(), v=pools["v"].data_ptr(), k_scale=scales["k"].data_ptr(),
                           v_scale=scales["v"].data_ptr(), table=table.data_ptr(), n_pages=total, page=page,
                           n_kv_heads=Hkv, head_dim=D, table_ld=2), "err": torch.zeros(1, dtype=torch.int32, device=cuda)}
    g = torch.Generator().manual_seed(4)
    new = torch.randn(150, 2, Hkv, D, generator=g).half().to(cuda)
    append(c, new, [150], [150])
    for n in (1, 150):
        q = torch.randn(n, Hkv * D, generator=g).half().to(cuda)
        out = torch.zeros_like(q)
        run_kv8(c, q, [n], [150], Hkv, out)
        # the same tokens in a small pool
        small = make_cache(cuda, 1, [150], Hkv, D, page)
        append(small, new, [150], [150])
        want = torch.zeros_like(q)
        run_kv8(small, q, [n], [150], Hkv, want)
        assert torch.equal(out, want) and float(out.abs().max()) > 0
    assert int(c["err"]) == 0


# ---------------------------------------------------------------- beam selection


def run_select(logits, cum, finished, eos, *, in_place=False):
    """logits [B, K, V] (strided rows allowed)."""
    import pkc
    import torch
    B, K, V = logits.shape
    dev = logits.device
    score = cum.clone() if in_place else torch.full((B, K), float("nan"), device=dev)
    done = finished.clone() if in_place else torch.full((B, K), 9, dtype=torch.uint8, device=dev)
    parent, token = (torch.full((B, K), -3, dtype=torch.int32, device=dev) for _ in range(2))
    names = {torch.float16: "f16", torch.bfloat16: "bf16", torch.float32: "f32"}
    pkc.beam_select(logits.data_ptr(), score.data_ptr() if in_place else cum.data_ptr(),
                    done.data_ptr() if in_place else finished.data_ptr(), B, K, V, eos=eos, dtype=names[logits.dtype],
                    score=score.data_ptr(), parent=parent.data_ptr(), token=token.data_ptr(),
                    finished_out=done.data_ptr(), ld=logits.stride(1), stream=stream())
    torch.cuda.synchronize()
    return score, parent, token, done


def check_select(logits, cum, finished, eos, **kw):
    import decode_ref
    import torch
    score, parent, token, done = run_select(logits, cum, finished, eos, **kw)
    rs, rp, rt, rd = decode_ref.beam_select(logits, cum, finished.bool(), eos)
    assert torch.equal(parent.long(), rp)
    assert torch.equal(token.long(), rt)
    assert torch.equal(done.bool(), rd) and (done <= 1).all()
    fin = torch.isfinite(rs)
    assert torch.equal(torch.isfinite(score), fin) and (score[~fin] == rs[~fin].float()).all()
    # exponentials within 2^-22 of their values: so is their sum's logarithm; one rounding to f32
    assert ((score.double() - rs)[fin].abs() <= 2.0 ** -21 + rs[fin].abs() * 2.0 ** -24 * 1.01).all()


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 1025), (3, 8, 33), (2, 5, 4099), (5, 8, 8193), (1, 2, 65537),
                                   (2, 16, 9001), (1, 32, 20000), (4, 10, 7), (2, 32, 2)])
def test_beam_select(cuda, dtype, B, K, V):
    import torch
    g = torch.Generator().manual_seed(B * 100 + K + V)
    dt = getattr(torch, dtype)
    store = torch.full((B, K, V + 5), float("nan"), dtype=dt, device=cuda)
    store[..., :V] = (torch.randn(B, K, V, generator=g) * 3).to(dt).to(cuda)
    logits = store[..., :V]
    cum = (torch.randn(B, K, generator=g) * 2 - 10).to(cuda)
    finished = (torch.rand(B, K, generator=g) < 0.2).to(torch.uint8).to(cuda)
    for eos in {0, V // 2, V - 1}:
        check_select(logits, cum, finished, eos)
        check_select(logits, cum, torch.zeros_like(finished), eos, in_place=True)


@pytest.mark.parametrize("B,K,V", [(2, 4, 700), (1, 8, 9000), (1, 2, 40000), (1, 32, 8193)])
def test_beam_select_ties(cuda, B, K, V):
    """Logits of a few values (many exact ties, within a row and, with equal
    scores, between rows whose logits are the same): the lowest index wins."""
    import torch
    g = torch.Generator().manual_seed(V)
    row = torch.randint(-2, 3, (B, 1, V), generator=g).float()
    logits = row.expand(B, K, V).contiguous().to(cuda)
    cum = torch.zeros(B, K, device=cuda)
    no = torch.zeros(B, K, dtype=torch.uint8, device=cuda)
    _, parent, token, _ = run_select(logits, cum, no, V - 1)
    flat = logits.double().flatten(1)
    at = torch.sort(flat, dim=1, descending=True, stable=True)[1][:, :K]
    assert torch.equal(parent.long(), at // V) and torch.equal(token.long(), at % V)
    # the same rows on 16-byte boundaries, and in 16 bits
    for dt, pad in ((torch.float32, (-V) % 4), (torch.float16, (-V) % 8), (torch.float16, 1)):
        wide = torch.zeros(B, K, V + pad, dtype=dt, device=cuda)
        wide[..., :V] = logits
        _, parent, token, _ = run_select(wide[..., :V], cum, no, V - 1)
        assert torch.equal(parent.long(), at // V) and torch.equal(token.long(), at % V)
    # constant rows: tokens 0 .. of beam 0
    _, parent, token, _ = run_select(torch.full_like(logits, -3.5), cum, no, V - 1)
    want = torch.arange(K, device=cuda).expand(B, K)
    assert torch.equal(parent.long(), want // V) and torch.equal(token.long(), want % V)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("B,K,V,live", [(2, 5, 50736, 3), (1, 32, 9001, 20), (3, 8, 8193, 8), (2, 16, 700, 1),
                                        (1, 4, 4096, 0)])
@pytest.mark.parametrize("mask", ["lowest", "-inf", "-1e4"])
def test_beam_select_masked_vocabulary(cuda, dtype, B, K, V, live, mask):
    """A mask that leaves a row few tokens, fewer than K among them: the others
    are all alike, and the lowest of them fill the places."""
    import torch
    g = torch.Generator().manual_seed(V + live)
    dt = getattr(torch, dtype)
    value = {"lowest": torch.finfo(dt).min, "-inf": float("-inf"), "-1e4": -1e4}[mask]
    logits = torch.full((B, K, V), value, dtype=dt)
    for b in range(B):
        for k in range(K):
            at = torch.randperm(V, generator=g)[:live]
            logits[b, k, at] = torch.randn(live, generator=g).to(dt)
    cum = torch.randn(B, K, generator=g) - 10
    check_select(logits.to(cuda), cum.to(cuda), torch.zeros(B, K, dtype=torch.uint8, device=cuda), V - 1)


def test_beam_select_zeros_of_either_sign(cuda):
    """-0 and +0 are the same logit and the same score: the lowest index wins."""
    import torch
    B, K, V = 1, 4, 300
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        logits = torch.zeros(B, K, V, dtype=dt, device=cuda)
        logits[..., ::2] = -0.0
        cum = torch.zeros(B, K, device=cuda)
        cum[:, 0] = -0.0
        no = torch.zeros(B, K, dtype=torch.uint8, device=cuda)
        _, parent, token, _ = run_select(logits, cum, no, V - 1)
        assert (parent == 0).all() and torch.equal(token.long(), torch.arange(K, device=cuda).expand(B, K))
        # finished hypotheses with scores of either sign: the lower beam first
        score, parent, token, _ = run_select(logits, cum, torch.ones_like(no), 7)
        assert torch.equal(parent.long(), torch.arange(K, device=cuda).expand(B, K)) and (token == 7).all()
        assert (score == 0).all()


def test_beam_select_sorted_rows(cuda):
    """Ascending and descending rows, and the largest values all in one
    thread's share."""
    import torch
    B, K, V = 3, 32, 8192
    logits = torch.zeros(B, K, V, device=cuda)
    logits[0] = torch.arange(V, device=cuda) * 1e-3
    logits[1] = torch.arange(V, device=cuda).flip(0) * 1e-3
    logits[2] = torch.where(torch.arange(V, device=cuda) % 256 == 7, torch.arange(V, device=cuda) * 1e-3 + 50, 0.0)
    logits = logits + torch.arange(K, device=cuda)[None, :, None] * 1e-5
    cum = -torch.arange(K, device=cuda).float().expand(B, K).contiguous() * 1e-4
    check_select(logits, cum, torch.zeros(B, K, dtype=torch.uint8, device=cuda), 5)


@pytest.mark.parametrize("V", [50, 9000])
def test_beam_select_dead_rows(cuda, V):
    """-inf scores (the first step), -inf logits (masked tokens), rows with a
    NaN, with +inf or with nothing but -inf, and a NaN score."""
    import torch
    B, K = 6, 4
    g = torch.Generator().manual_seed(V)
    logits = torch.randn(B, K, V, generator=g).to(cuda)
    cum = (torch.randn(B, K, generator=g)).to(cuda)
    inf = float("inf")
    cum[0, 1:] = -inf                      # the first step
    cum[1] = -inf                          # nothing left
    logits[2, :, 3:] = -inf                # three tokens allowed
    logits[3, 0, 7] = float("nan")
    logits[3, 1, V - 1] = inf
    logits[3, 2] = -inf
    cum[4, 2] = float("nan")
    fin = torch.zeros(B, K, dtype=torch.uint8, device=cuda)
    fin[5] = 1                             # all finished
    fin[3, 3] = 1
    for eos in (0, 2, V - 1):
        check_select(logits, cum, fin, eos)


def test_beam_select_close_scores(cuda):
    """Hypotheses whose scores differ by less than a step of f32 at their size
    come out in the order of their exact scores."""
    import torch
    B, K, V = 16, 8, 2000
    g = torch.Generator().manual_seed(8)
    row = torch.randn(B, 1, V, generator=g).expand(B, K, V).clone()
    row[:, :, 0] = 30.0  # the token that every row takes, nearly all the weight
    # the rows differ in a far lower logit: sums differ by 1e-4 .. relative
    row[:, :, 1] = 20.0 + torch.rand(B, K, generator=g)
    cum = torch.full((B, K), -1000.0)
    check_select(row.to(cuda), cum.to(cuda), torch.zeros(B, K, dtype=torch.uint8, device=cuda), V - 1)


# ---------------------------------------------------------------- reordering


@pytest.mark.parametrize("K", [1, 2, 4, 5, 8, 16, 32])
@pytest.mark.parametrize("row_bytes,stride,align", [(4096, 4096, 0), (4100, 4112, 0), (37, 37, 1), (640, 648, 0), (1, 3, 2)])
def test_beam_reorder(cuda, K, row_bytes, stride, align):
    import pkc
    import torch
    B, O = 3, 2
    g = torch.Generator().manual_seed(K + row_bytes)
    outer = B * K * stride + 5 * (stride % 2)
    buf = torch.randint(0, 256, (align + O * outer + 64,), generator=g, dtype=torch.uint8).to(cuda)
    parent = torch.randint(0, K, (B, K), generator=g, dtype=torch.int32)
    parent[0] = torch.arange(K, dtype=torch.int32).flip(0)
    parent = parent.to(cuda)
    for lens in (None, torch.tensor([3, 0, 100000], dtype=torch.int32, device=cuda)):
        want = buf.clone()
        for o in range(O):
            for b in range(B):
                live = row_bytes if lens is None else min(row_bytes, int(lens[b]) * 11)
                rows = torch.as_strided(buf, (K, live), (stride, 1), align + o * outer + b * K * stride)
                torch.as_strided(want, (K, live), (stride, 1), align + o * outer + b * K * stride).copy_(rows[parent[b].long()])
        got = buf.clone()
        pkc.beam_reorder(got.data_ptr() + align, parent.data_ptr(), B, K, row_bytes=row_bytes, row_stride=stride, n_outer=O,
                         outer_stride=outer, lens=0 if lens is None else lens.data_ptr(), unit_bytes=11, stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_beam_reorder_bad_parent(cuda):
    """A parent outside [0, K) is reported and that row stays."""
    import pkc
    import torch
    x = torch.arange(4, dtype=torch.float32, device=cuda).repeat_interleave(8).view(4, 8).clone()
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    parent = torch.tensor([[3, 4, -1, 0]], dtype=torch.int32, device=cuda)
    pkc.beam_reorder(x.data_ptr(), parent.data_ptr(), 1, 4, row_bytes=32, err=err.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert int(err) == 110 and x[:, 0].tolist() == [3.0, 1.0, 2.0, 0.0]


@pytest.mark.parametrize("K", [1, 3, 8, 16, 32])
@pytest.mark.parametrize("length,page,D", [(0, 16, 64), (5, 16, 64), (64, 32, 128), (77, 32, 128), (16, 16, 64), (130, 128, 64)])
def test_kv8_reorder(cuda, K, length, page, D):
    """After it, each sequence reads what its parent's read before, each page
    that fills is its sequence's own, and entries behind it are as before."""
    import pkc
    import torch
    B, Hkv = 2, 2
    lens = [length, max(0, length - 3)] if length % page else [length, length]
    per = [n for n in lens for _ in range(K)]
    c = make_cache(cuda, B * K, [n + page for n in per], Hkv, D, page, seed=K)
    g = torch.Generator().manual_seed(K + length)
    for x in "kv":
        c[x].copy_(torch.randint(0, 120, c[x].shape, generator=g, dtype=torch.uint8))
        c[x + "_scale"].copy_(torch.exp2(torch.randint(-5, 6, c[x + "_scale"].shape, generator=g).float()))

    def dense(s):
        out = []
        for x in "kv":
            ids = c["table"][s, : -(-per[s] // page)].long()
            out.append(c[x][ids].transpose(1, 2).reshape(-1, Hkv, D)[: per[s]].clone())
            out.append(c[x + "_scale"][ids].clone())
        return out

    before = [dense(s) for s in range(B * K)]
    table = c["table"].clone()
    parent = torch.randint(0, K, (B, K), generator=g, dtype=torch.int32).to(cuda)
    ln = torch.tensor(per, dtype=torch.int32, device=cuda)
    pkc.kv8_reorder(c["c"], parent.data_ptr(), ln.data_ptr(), B, K, err=c["err"].data_ptr(), stream=stream())
    torch.cuda.synchronize()
    assert int(c["err"]) == 0
    for s in range(B * K):
        src = s // K * K + int(parent.flatten()[s])
        for a, b in zip(dense(s), before[src]):
            assert torch.equal(a, b)
        full = per[s] // page
        assert torch.equal(c["table"][s, full:], table[s, full:])


def test_kv8_reorder_refuses_on_the_device(cuda):
    """Uneven lengths, a shared page to fill, a bad parent or page: reported,
    and nothing of that item moves."""
    import pkc
    import torch
    for what in ("lens", "shared", "parent", "page"):
        c = make_cache(cuda, 4, [20] * 4, 1, 64, 16, fill=1)
        for s in range(4):
            for p in c["table"][s, :2].tolist():
                c["k"][p] = 10 * s + 1
        lens, parent = torch.full((4,), 20, dtype=torch.int32, device=cuda), torch.tensor([1, 0, 1, 0], dtype=torch.int32, device=cuda)
        if what == "lens":
            lens[3] = 19
        elif what == "shared":
            c["table"][3, 1] = c["table"][2, 1]
        elif what == "parent":
            parent[2] = 2
        else:
            c["table"][2, 1] = 1 << 20
        pool, table = c["k"].clone(), c["table"].clone()
        pkc.kv8_reorder(c["c"], parent.data_ptr(), lens.data_ptr(), 2, 2, err=c["err"].data_ptr(), stream=stream())
        torch.cuda.synchronize()
        assert int(c["err"]) == 110, what
        assert torch.equal(c["table"][2:], table[2:])
        assert torch.equal(c["table"][:2, 0].flip(0), table[:2, 0])  # the other item moved
        own = [p for p in table[2:].flatten().tolist() if 0 <= p < c["total"]]
        assert torch.equal(c["k"][own], pool[own])


# ---------------------------------------------------------------- several at once, captured, other streams


def test_small_workspaces_do_not_overlap(cuda):
    """Two calls on two streams at once, each with its own workspace, give what
    each gives alone."""
    import pkc
    import torch
    H, D, t = 8, 64, 9000
    g = torch.Generator().manual_seed(21)
    args = []
    for i in range(2):
        q = torch.randn(1, H * D, generator=g).half().to(cuda)
        kv = torch.randn(t, 2, H, D, generator=g).half().to(cuda)
        n = pkc.cross_attention_workspace(1, 1, t, H, H, D)
        assert n > 0  # the joined form
        args.append(dict(q=q, kv=kv, ws=workspace(n, cuda), out=torch.zeros(1, H * D, dtype=torch.float16, device=cuda),
                         q_off=offsets([1], cuda), kv_off=torch.zeros(1, dtype=torch.int32, device=cuda),
                         kv_len=torch.full((1,), t, dtype=torch.int32, device=cuda)))

    def call(a, out, st):
        pkc.cross_attention(a["q"].data_ptr(), a["kv"].data_ptr(), a["kv"][:, 1].data_ptr(), a["q_off"].data_ptr(),
                            a["kv_off"].data_ptr(), a["kv_len"].data_ptr(), 1, H, H, D, q_rows=1, kv_rows=t, max_q=1,
                            max_kv=t, ldk=2 * H * D, ldv=2 * H * D, bf16=False, out=out.data_ptr(),
                            workspace=a["ws"].data_ptr(), workspace_bytes=a["ws"].numel(), stream=st)

    want = []
    for a in args:
        o = torch.zeros_like(a["out"])
        call(a, o, stream())
        torch.cuda.synchronize()
        want.append(o)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for a, st in zip(args, s):
            call(a, a["out"], st.cuda_stream)
    torch.cuda.synchronize()
    for a, w in zip(args, want):
        assert torch.equal(a["out"], w)


class Decoder:
    """A small attention decoder (random weights, 16-bit) run by the library's
    operators: self attention over the 8-bit cache, cross attention to encoder
    states, logits, selection, reordering."""

    def __init__(self, cuda, B, K, page, steps, dt, *, layers=2, H=4, Hkv=2, D=64, V=211, seed=3):
        import pkc
        import torch
        self.B, self.K, self.page, self.steps, self.L, self.H, self.Hkv, self.D, self.V = B, K, page, steps, layers, H, Hkv, D, V
        self.dev, self.dt, self.eos = cuda, dt, 7
        d = self.d = H * D
        g = torch.Generator().manual_seed(seed)
        mk = lambda *s, scale: (torch.randn(*s, generator=g) * scale).to(dt).to(cuda)  # noqa: E731
        self.embed = mk(V, d, scale=1.0)
        self.w = [dict(qkv=mk(d, d + 2 * Hkv * D, scale=d ** -0.5), o=mk(d, d, scale=d ** -0.5), cq=mk(d, d, scale=d ** -0.5),
                       co=mk(d, d, scale=d ** -0.5)) for _ in range(layers)]
        self.head = mk(d, V, scale=3 * d ** -0.5)
        self.enc_len = [40, 3, 77, 0, 25][:B]
        M = sum(self.enc_len)
        self.enc = [mk(M, 2, H * D, scale=1.0) for _ in range(layers)]
        self.kv_off = offsets(self.enc_len, cuda)[:-1].contiguous()
        self.kv_len = torch.tensor(self.enc_len, dtype=torch.int32, device=cuda)
        S = B * K
        self.caches = [make_cache(cuda, S, [steps + 1] * S, Hkv, D, page, seed=i) for i in range(layers)]
        self.one = offsets([1] * S, cuda)
        self.beams = offsets([K] * B, cuda)
        self.lens = torch.zeros(S, dtype=torch.int32, device=cuda)
        self.token = torch.zeros(B, K, dtype=torch.int32, device=cuda)
        self.parent = torch.zeros(B, K, dtype=torch.int32, device=cuda)
        self.cum = torch.zeros(B, K, device=cuda)
        self.cum[:, 1:] = float("-inf")
        self.done = torch.zeros(B, K, dtype=torch.uint8, device=cuda)
        self.history = torch.full((S, steps), -1, dtype=torch.int32, device=cuda)
        self.step_at = torch.zeros(1, dtype=torch.int64, device=cuda)
        self.seen = []
        self.ws = workspace(max(pkc.cross_attention_workspace(B, K, 77, H, H, D), pkc.kv8_attention_workspace(
            self.caches[0]["c"], S, 1, steps, H)), cuda)

    def step(self):
        import pkc
        import torch
        B, K, S, H, D, d = self.B, self.K, self.B * self.K, self.H, self.D, self.d
        bf, st = self.dt == torch.bfloat16, stream()
        self.seen = []
        self.lens += 1
        x = self.embed[self.token.flatten().long()].float()
        for i, (w, c) in enumerate(zip(self.w, self.caches)):
            qkv = torch.nn.functional.layer_norm(x, (d,)).to(self.dt) @ w["qkv"]
            n = self.Hkv * D
            ld = qkv.stride(0)
            pkc.kv8_append(c["c"], qkv[:, d:].data_ptr(), qkv[:, d + n:].data_ptr(), self.one.data_ptr(), self.lens.data_ptr(), S,
                           rows=S, max_new=1, ldk=ld, ldv=ld, bf16=bf, err=c["err"].data_ptr(), stream=st)
            a = torch.empty(S, d, dtype=self.dt, device=self.dev)
            pkc.kv8_attention(c["c"], qkv.data_ptr(), self.one.data_ptr(), self.lens.data_ptr(), S, H, q_rows=S, max_q=1,
                              max_len=self.steps, ldq=ld, bf16=bf, out=a.data_ptr(), workspace=self.ws.data_ptr(),
                              workspace_bytes=self.ws.numel(), err=c["err"].data_ptr(), stream=st)
            x = x + (a @ w["o"]).float()
            cq = torch.nn.functional.layer_norm(x, (d,)).to(self.dt) @ w["cq"]
            ca = torch.empty(S, d, dtype=self.dt, device=self.dev)
            e = self.enc[i]
            pkc.cross_attention(cq.data_ptr(), e.data_ptr(), e[:, 1].data_ptr(), self.beams.data_ptr(), self.kv_off.data_ptr(),
                                self.kv_len.data_ptr(), B, H, H, D, q_rows=S, kv_rows=e.shape[0], max_q=K, max_kv=77,
                                ldk=2 * d, ldv=2 * d, bf16=bf, out=ca.data_ptr(), workspace=self.ws.data_ptr(),
                                workspace_bytes=self.ws.numel(), err=c["err"].data_ptr(), stream=st)
            self.seen += [qkv, a, cq, ca]
            x = x + (ca @ w["co"]).float()
        logits = torch.nn.functional.layer_norm(x, (d,)).to(self.dt).float() @ self.head.float()
        self.seen += [logits, self.cum.clone(), self.done.clone()]
        pkc.beam_select(logits.data_ptr(), self.cum.data_ptr(), self.done.data_ptr(), B, K, self.V, eos=self.eos,
                        score=self.cum.data_ptr(), parent=self.parent.data_ptr(), token=self.token.data_ptr(),
                        finished_out=self.done.data_ptr(), stream=st)
        for c in self.caches:
            pkc.kv8_reorder(c["c"], self.parent.data_ptr(), self.lens.data_ptr(), B, K, err=c["err"].data_ptr(), stream=st)
        pkc.beam_reorder(self.history.data_ptr(), self.parent.data_ptr(), B, K, row_bytes=4 * self.steps, err=self.caches[0]["err"].data_ptr(),
                         stream=st)
        self.history.scatter_(1, self.step_at.expand(S, 1), self.token.view(S, 1))
        self.step_at += 1
        # (the operators are done with these when the stream is; keep them until then)
        self.keep = (x, logits)


@pytest.mark.parametrize("bf16,B,K,page,steps", [(False, 3, 4, 16, 37), (True, 4, 8, 32, 20), (False, 5, 1, 16, 18)])
def test_decoder_beam_search(cuda, bf16, B, K, page, steps):
    """A whole beam search: after every step each operator's output is checked
    against the 64-bit restatement of the same step, whose caches and
    hypotheses follow their own history (dense, copied at each reordering)."""
    import decode_ref
    import torch
    dt = torch.bfloat16 if bf16 else torch.float16
    m = Decoder(cuda, B, K, page, steps, dt)
    S, H, Hkv, D, d = B * K, m.H, m.Hkv, m.D, m.d
    # the restatement: for each layer and sequence a cache of its own with identity pages
    n_pg = -(-(steps + 1) // page)
    refs = [[decode_ref.RefCache(n_pg, Hkv, page, D) for _ in range(S)] for _ in range(m.L)]
    texts = [[] for _ in range(S)]
    for t in range(1, steps + 1):
        m.step()
        torch.cuda.synchronize()
        assert all(int(c["err"]) == 0 for c in m.caches)
        for i in range(m.L):
            qkv, a, cq, ca = m.seen[4 * i: 4 * i + 4]
            for s in range(S):
                r = refs[i][s]
                r.append(list(range(n_pg)), qkv[s, d:].double().view(1, 2, Hkv, D).cpu(), t)
                k, v = (y.to(cuda) for y in r.dense(list(range(n_pg)), t))
                o, A, S_ = decode_ref.attention(qkv[s, :d].double().view(1, H, D), k, v, D ** -0.5, True)
                tol = decode_ref.attention_tolerance(o, A, S_, float(v.abs().max()), t, D, dt, torch.float16)
                assert ((a[s].double().view(1, H, D) - o).abs() <= tol).all(), (t, i, s)
            for b in range(B):
                e = m.enc[i][int(m.kv_off[b]): int(m.kv_off[b]) + m.enc_len[b]].double().view(-1, 2, H, D)
                o, A, S_ = decode_ref.attention(cq[b * K:(b + 1) * K].double().view(K, H, D), e[:, 0], e[:, 1], D ** -0.5, False)
                v_max = float(e[:, 1].abs().max()) if m.enc_len[b] else 0.0
                tol = decode_ref.attention_tolerance(o, A, S_, v_max, m.enc_len[b], D, dt, dt)
                assert ((ca[b * K:(b + 1) * K].double().view(K, H, D) - o).abs() <= tol).all(), (t, i, b)
        logits, cum, done = m.seen[-3:]
        rs, rp, rt, rd = decode_ref.beam_select(logits.view(B, K, -1), cum, done.bool(), m.eos)
        assert torch.equal(m.parent.long(), rp) and torch.equal(m.token.long(), rt) and torch.equal(m.done.bool(), rd)
        src = [b * K + int(rp[b, k]) for b in range(B) for k in range(K)]
        import copy
        refs = [[copy.deepcopy(layer[j]) for j in src] for layer in refs]
        texts = [texts[j] + [int(rt.flatten()[s])] for s, j in enumerate(src)]
        assert m.history[:, :t].tolist() == texts
    assert len({tuple(x) for x in texts}) > 1 or K == 1


def test_decoder_step_captured_and_replayed(cuda):
    """One captured step replayed (lengths, tokens and tables move on the
    device) takes the path of the eager steps, bit for bit, also on another
    stream."""
    import torch
    runs = []
    for how in ("eager", "graph", "side"):
        m = Decoder(cuda, 3, 4, 16, 24, torch.float16)
        if how == "graph":
            # (a warm-up step outside the capture, on a decoder of its own)
            Decoder(cuda, 3, 4, 16, 24, torch.float16).step()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                m.step()
            for _ in range(24):
                g.replay()
        elif how == "side":
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                for _ in range(24):
                    m.step()
        else:
            for _ in range(24):
                m.step()
        torch.cuda.synchronize()
        assert all(int(c["err"]) == 0 for c in m.caches)
        runs.append(m)
    for m in runs[1:]:
        assert torch.equal(m.history, runs[0].history) and torch.equal(m.cum, runs[0].cum)
        for c, e in zip(m.caches, runs[0].caches):
            assert torch.equal(c["table"], e["table"]) and torch.equal(c["k"], e["k"]) and torch.equal(c["v"], e["v"])


def test_the_first_call_may_be_captured(cuda):
    """In a new process: the first call of every operator under capture, then
    replayed."""
    import os
    import subprocess
    import sys
    code = """
import sys
sys.path[:0] = [%r, %r]
import torch
import test_decode_gpu as T
dev = torch.device("cuda:0")
m, e = (T.Decoder(dev, 2, 3, 16, 6, torch.bfloat16, seed=9) for _ in range(2))
many = T.make_cache(dev, 1, [200], 2, 64, 32)
kv = torch.randn(200, 2, 2, 64, device=dev).half()
out = torch.zeros(200, 128, dtype=torch.float16, device=dev)
no, ln = T.offsets([200], dev), torch.full((1,), 200, dtype=torch.int32, device=dev)
zero = torch.zeros(1, dtype=torch.int32, device=dev)
import pkc
ws = T.workspace(max(1, pkc.kv8_attention_workspace(many["c"], 1, 200, 200, 2), pkc.cross_attention_workspace(1, 200, 200, 2, 2, 64)), dev)
torch.zeros(8, 8, device=dev).half() @ torch.zeros(8, 8, device=dev).half()  # torch's own product needs a first call
torch.zeros(8, 8, device=dev) @ torch.zeros(8, 8, device=dev)
torch.zeros(8, 8, device=dev).bfloat16() @ torch.zeros(8, 8, device=dev).bfloat16()
def prompt(st):
    pkc.kv8_append(many["c"], kv.data_ptr(), kv[:, 1].data_ptr(), no.data_ptr(), ln.data_ptr(), 1, rows=200, max_new=200,
                   ldk=256, ldv=256, bf16=False, err=many["err"].data_ptr(), stream=st)
    pkc.kv8_attention(many["c"], kv.data_ptr(), no.data_ptr(), ln.data_ptr(), 1, 2, q_rows=200, max_q=200, max_len=200,
                      ldq=256, bf16=False, out=out.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                      err=many["err"].data_ptr(), stream=st)
    pkc.cross_attention(out.data_ptr(), kv.data_ptr(), kv[:, 1].data_ptr(), no.data_ptr(), zero.data_ptr(), ln.data_ptr(), 1, 2, 2, 64,
                        q_rows=200, kv_rows=200, max_q=200, max_kv=200, ldk=256, ldv=256, bf16=False, out=res.data_ptr(),
                        workspace=ws.data_ptr(), workspace_bytes=ws.numel(), err=many["err"].data_ptr(), stream=st)
res = torch.zeros_like(out)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    m.step()
    prompt(T.stream())
for _ in range(6):
    g.replay()
torch.cuda.synchronize()
a = res.clone()
for _ in range(6):
    e.step()
prompt(T.stream())
torch.cuda.synchronize()
assert int(many["err"]) == 0 and torch.equal(a, res) and float(a.abs().max()) > 0
assert torch.equal(m.history, e.history) and torch.equal(m.cum, e.cum)
print("captured ok")
""" % (os.path.dirname(os.path.abspath(__file__)), os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "parakeet.cpp_b200", "python"))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured ok" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]


def test_a_prompt_then_steps_equals_one_pass(cuda):
    """Appending and attending in chunks (the many-row form), then token by
    token, gives the rows that one pass over all tokens gives, as near as the
    page scales allow: the cache of a page that grew is rounded again, so the
    pages here are filled with values of one size."""
    import torch
    H, Hkv, D, page, n = 4, 2, 64, 32, 300
    g = torch.Generator().manual_seed(31)
    sign = (torch.randint(0, 2, (n, 2, Hkv, D), generator=g) * 2 - 1).float()
    new = sign * (1 + torch.randint(0, 8, (n, 2, Hkv, D), generator=g) / 8)
    new[:, :, :, 0] = 1.875  # the largest, in every token: one scale, and every value an e4m3 value
    new = new.half().to(cuda)
    q = torch.randn(n, H * D, generator=g).half().to(cuda)
    whole = make_cache(cuda, 1, [n], Hkv, D, page)
    append(whole, new, [n], [n])
    want = torch.zeros_like(q)
    run_kv8(whole, q, [n], [n], H, want)
    parts = make_cache(cuda, 1, [n], Hkv, D, page, seed=5)
    out = torch.zeros_like(q)
    at = 0
    for size in (150, 3, 1, 1, 60, 20, 1, 64):
        append(parts, new[at:at + size], [size], [at + size])
        o = torch.zeros_like(q[at:at + size])
        run_kv8(parts, q[at:at + size].contiguous(), [size], [at + size], H, o)
        out[at:at + size] = o
        at += size
    assert at == n
    # the same sums in another order: f16 probabilities, one rounding of the output
    assert ((out.double() - want.double()).abs() <= 2 * (2.0 ** -11 + 2.0 ** -11) * 1.875).all()


def test_negative_and_zero_scale(cuda):
    """scale may be negative or zero (even weights)."""
    for scale in (-0.2, 0.0):
        check_cross(cuda, [3, 140], [50, 90], 4, 2, 64, False, scale=scale)
