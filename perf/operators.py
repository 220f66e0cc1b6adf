"""What the operators of an attention decoder over the encoder's output cost: cross attention, the 8-bit key/value cache and the attention
over it, beam selection and the reordering of states. Each case is one call as a beam search or a rescoring pass makes it.

`run` computes a case in plain torch operations, or, where `own` is true, through the library's kernel-level entry points."""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one clip of 35 s (437 frames), one hypothesis, one token: what a single request waits for
        {"name": "cross: step, one clip", "op": "cross", "B": 1, "qmin": 1, "qmax": 1, "tmin": 437, "tmax": 437, "H": 8, "Hkv": 8, "D": 128, "dtype": "f16"},
        # one decoder step of a batch of 64 clips of 2 to 35 s with 8 hypotheses each
        {"name": "cross: step, 64 clips x 8", "op": "cross", "B": 64, "qmin": 8, "qmax": 8, "tmin": 25, "tmax": 437, "H": 8, "Hkv": 8, "D": 128, "dtype": "bf16"},
        # rescoring of 8 hypotheses of up to 48 tokens a clip, clips of 20 to 120 s
        {"name": "cross: scoring", "op": "cross", "B": 64, "qmin": 130, "qmax": 384, "tmin": 250, "tmax": 1500, "H": 8, "Hkv": 8, "D": 128, "dtype": "f16"},
        # the write of one token's keys and values for 64 clips x 8 hypotheses
        {"name": "append: step, 512 beams", "op": "append", "S": 512, "nmin": 1, "nmax": 1, "omin": 0, "omax": 447, "Hkv": 8, "D": 128, "page": 32, "dtype": "bf16"},
        # prompts (earlier transcript) of uneven length onto caches that hold some tokens already
        {"name": "append: prompts", "op": "append", "S": 64, "nmin": 1, "nmax": 1024, "omin": 0, "omax": 1000, "Hkv": 8, "D": 64, "page": 64, "dtype": "f16"},
        # one decoder step of 64 clips x 8 hypotheses over their own tokens
        {"name": "kv8: step, 512 beams", "op": "kv8", "S": 512, "nmin": 1, "nmax": 1, "lmin": 1, "lmax": 448, "H": 8, "Hkv": 8, "D": 128, "page": 32, "dtype": "bf16"},
        # one step over very long contexts (hours of transcript), shared key heads
        {"name": "kv8: step, long", "op": "kv8", "S": 8, "nmin": 1, "nmax": 1, "lmin": 9001, "lmax": 131071, "H": 16, "Hkv": 2, "D": 128, "page": 64, "dtype": "f16"},
        # a chunk of a prompt over what the cache holds already
        {"name": "kv8: chunk", "op": "kv8", "S": 8, "nmin": 100, "nmax": 256, "lmin": 300, "lmax": 16384, "H": 16, "Hkv": 4, "D": 64, "page": 64, "dtype": "bf16"},
        # selection for one clip, 4 hypotheses, the small vocabulary
        {"name": "select: one clip", "op": "select", "B": 1, "K": 4, "V": 1025, "dtype": "f32"},
        # selection for 64 clips x 8 hypotheses, the large vocabulary
        {"name": "select: 64 clips x 8", "op": "select", "B": 64, "K": 8, "V": 8193, "dtype": "f32"},
        # dense f16 states (4 layers of keys and of values, 100 tokens so far) follow their hypotheses
        {"name": "reorder: dense", "op": "rows", "B": 64, "K": 8, "outer": 8, "cap": 128, "live": 100, "unit": 1024, "dtype": "f16"},
        # the 8-bit cache follows its hypotheses: tables, and the pages being filled
        {"name": "reorder: pages", "op": "pages", "B": 64, "K": 8, "lmin": 1, "lmax": 448, "Hkv": 8, "D": 128, "page": 32},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cross", "cross", "append", "kv8", "kv8", "select", "rows", "pages"])
    D = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    H = Hkv * rng.choice([1, 2, 4]) if Hkv < 8 else 8
    dt = rng.choice(["f16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "cross":
        B, T = _log(rng, 1, 64), _log(rng, 1, 45000)
        B = max(1, min(B, 96000 // T))
        q = _log(rng, 1, 384)
        q = max(1, min(q, 6_000_000 // (B * T)))
        return {"op": op, "B": B, "qmin": max(1, q // 3), "qmax": q, "tmin": rng.choice([0, max(1, T // 4), T]), "tmax": T, "H": H, "Hkv": Hkv, "D": D, "dtype": dt}
    if op == "append":
        S = _log(rng, 1, 512)
        n = rng.choice([1, _log(rng, 1, max(1, 32768 // S))])
        return {"op": op, "S": S, "nmin": rng.choice([0, 1, n]), "nmax": n, "omin": 0, "omax": _log(rng, 1, max(1, min(1000, 200000 // S))), "Hkv": Hkv, "D": D, "page": page, "dtype": dt}
    if op == "kv8":
        S = _log(rng, 1, 512)
        L = _log(rng, 1, max(448, min(131071, 400000 // S)))
        n = rng.choice([1, 1, min(L, _log(rng, 1, 256))])
        n = max(1, min(n, 16_000_000 // (S * L)))
        return {"op": op, "S": S, "nmin": max(1, n // 2), "nmax": n, "lmin": max(n, L // rng.choice([1, 4, 16])), "lmax": L, "H": H, "Hkv": Hkv, "D": D, "page": page, "dtype": dt}
    if op == "select":
        K, V = rng.choice([1, 2, 4, 5, 8, 10, 16]), _log(rng, 33, 65537)
        return {"op": op, "B": _log(rng, 1, max(1, min(64, 4_000_000 // (K * V)))), "K": K, "V": V, "dtype": rng.choice(["f32", "f32", "f16", "bf16"])}
    if op == "rows":
        K, unit, cap = rng.choice([2, 4, 5, 8, 16]), rng.choice([1, 3, 64, 640, 1024]), _log(rng, 1, 128)
        return {"op": op, "B": max(1, _log(rng, 1, 64) * 8 // max(8, K)), "K": K, "outer": rng.choice([1, 2, 8]), "cap": cap, "live": rng.randint(1, cap), "unit": unit, "dtype": rng.choice(["f16", "f32"])}
    K = rng.choice([2, 4, 5, 8, 16])
    return {"op": op, "B": max(1, _log(rng, 1, 64) * 8 // max(8, K)), "K": K, "lmin": 1, "lmax": _log(rng, 1, 448), "Hkv": Hkv, "D": D, "page": page}


def _lengths(n, lo, hi, salt):
    """n lengths in [lo, hi], the largest first: the same ones for every seed, so that a case's work is known."""
    r = random.Random("%d %d %d %s" % (n, lo, hi, salt))
    return [hi] + [r.randint(lo, hi) for _ in range(n - 1)]


def _sizes(c):
    op = c["op"]
    if op == "cross":
        return _lengths(c["B"], c["qmin"], c["qmax"], "q"), _lengths(c["B"], c["tmin"], c["tmax"], "t")
    if op == "append":
        n, old = _lengths(c["S"], c["nmin"], c["nmax"], "n"), _lengths(c["S"], c["omin"], c["omax"], "o")
        return n, [a + b for a, b in zip(n, old)]
    if op == "kv8":
        n, length = _lengths(c["S"], c["nmin"], c["nmax"], "n"), _lengths(c["S"], c["lmin"], c["lmax"], "l")
        return n, length
    return [], _lengths(c["B"], c["lmin"], c["lmax"], "l") if op == "pages" else []


def _offsets(lens, dev):
    t = torch.zeros(len(lens) + 1, dtype=torch.int32)
    t[1:] = torch.tensor(lens, dtype=torch.int32).cumsum(0)
    return t.to(dev)


def _cache(c, S, lens, g, dev):
    """A cache as earlier appends left it: pages in no order, codes of normal values, a scale for each page and head."""
    page, Hkv, D = c["page"], c["Hkv"], c["D"]
    need = [max(1, -(-n // page)) for n in lens]
    width, total = max(need), sum(need) + 3
    perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(S, width, dtype=torch.int32, device=dev)
    has = torch.arange(width, device=dev)[None, :] < torch.tensor(need, device=dev)[:, None]
    table.masked_scatter_(has, perm[: sum(need)])
    out = {"table": table, "n_pages": total, "width": width}
    for x in "kv":  # one page more than the cache has: see _plain_append
        out[x] = (torch.randn(total + 1, Hkv, page, D, generator=g, device=dev, dtype=torch.float16) * 110).clamp_(-448, 448).to(torch.float8_e4m3fn)
        out[x + "_scale"] = torch.exp2(torch.randint(-8, -5, (total + 1, Hkv), generator=g, device=dev).float())
    return out


def prepare(case, seed):
    c, dev = case, torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rnd = lambda *s, dtype=torch.float32: torch.randn(*s, generator=g, device=dev, dtype=dtype)  # noqa: E731
    s = {"case": c}
    a, b = _sizes(c)
    if c["op"] == "cross":
        dt = DTYPES[c["dtype"]]
        # keys and values as one projection leaves them: [frames, k | v]
        s.update(q=rnd(sum(a), c["H"], c["D"], dtype=dt), kv=rnd(max(1, sum(b)), 2, c["Hkv"], c["D"], dtype=dt), q_off=_offsets(a, dev), kv_off=_offsets(b, dev))
        s.update(kv_len=torch.tensor(b, dtype=torch.int32, device=dev), out=torch.zeros(sum(a), c["H"], c["D"], dtype=dt, device=dev))
    elif c["op"] == "append":
        dt = DTYPES[c["dtype"]]
        s.update(_cache(c, c["S"], b, g, dev), new_off=_offsets(a, dev), lens=torch.tensor(b, dtype=torch.int32, device=dev))
        # new values now and then larger than what a page's scale holds
        s["new"] = (rnd(max(1, sum(a)), 2, c["Hkv"], c["D"]) * torch.exp2(torch.randint(-1, 3, (max(1, sum(a)), 2, c["Hkv"], 1), generator=g, device=dev).float())).to(dt)
    elif c["op"] == "kv8":
        dt = DTYPES[c["dtype"]]
        s.update(_cache(c, c["S"], b, g, dev), q_off=_offsets(a, dev), lens=torch.tensor(b, dtype=torch.int32, device=dev))
        s.update(q=rnd(sum(a), c["H"], c["D"], dtype=dt), out=torch.zeros(sum(a), c["H"], c["D"], dtype=dt, device=dev))
    elif c["op"] == "select":
        B, K, V = c["B"], c["K"], c["V"]
        s.update(logits=(rnd(B * K, V) * 2.5).to(DTYPES[c["dtype"]]), cum=(rnd(B, K) * 3 - 20).sort(1, descending=True)[0].contiguous())
        s["finished"] = (torch.rand(B, K, generator=g, device=dev) < 0.1).to(torch.uint8)
        s.update(score=torch.zeros(B, K, device=dev), parent=torch.zeros(B, K, dtype=torch.int32, device=dev), token=torch.zeros(B, K, dtype=torch.int32, device=dev))
        s["done"] = torch.zeros(B, K, dtype=torch.uint8, device=dev)
    else:
        B, K = c["B"], c["K"]
        keep = torch.arange(K, device=dev).expand(B, K)
        s["parent"] = torch.where(torch.rand(B, K, generator=g, device=dev) < 0.4, keep, torch.randint(0, K, (B, K), generator=g, device=dev)).to(torch.int32)
        if c["op"] == "rows":
            s["state"] = rnd(c["outer"], B * K, c["cap"], c["unit"], dtype=DTYPES[c["dtype"]])
        else:
            lens = [n for n in b for _ in range(K)]
            s.update(_cache(c, B * K, lens, g, dev), lens=torch.tensor(lens, dtype=torch.int32, device=dev))
    return s


def _whole(s, *more):
    return {**{x: s[x][: s["n_pages"]] for x in ("k", "v", "k_scale", "v_scale")}, **{x: s[x] for x in more}}


# ---------------------------------------------------------------- plain forms


def _rows_of(off, n, total):
    """For each packed row its item and its place there."""
    item = torch.repeat_interleave(torch.arange(n, device=off.device), (off[1:] - off[:-1]).long(), output_size=total)
    return item, torch.arange(total, device=off.device) - off[:-1].long()[item]


def _padded(off, n, most, total):
    at = off[:-1].long()[:, None] + torch.arange(most, device=off.device)[None, :]
    return at.clamp_(max=max(0, total - 1))


def _attend(q, k, v, seen, item, pos, scale):
    """q [B, Q, Hkv, G, D], k / v [B, T, Hkv, D] in 32 bits, seen [B, Q, T] -> [rows, H, D]."""
    s = torch.einsum("bqhgd,bthd->bhgqt", q, k) * scale
    s.masked_fill_(~seen[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True) if s.shape[-1] else s.sum(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.einsum("bhgqt,bthd->bqhgd", p, v)
    return o.flatten(2, 3)[item, pos]


def _plain_cross(s):
    c, dev = s["case"], s["q"].device
    B, Q, T, Hkv = c["B"], c["qmax"], c["tmax"], c["Hkv"]
    total, G = s["q"].shape[0], c["H"] // c["Hkv"]
    item, pos = _rows_of(s["q_off"], B, total)
    q = s["q"][_padded(s["q_off"], B, Q, total)].float().unflatten(2, (Hkv, G))
    kv = s["kv"][_padded(s["kv_off"], B, T, s["kv"].shape[0])].float()
    seen = (torch.arange(T, device=dev)[None, :] < s["kv_len"][:, None])[:, None].expand(B, Q, T)
    return _attend(q, kv[:, :, 0], kv[:, :, 1], seen, item, pos, 1 / math.sqrt(c["D"])).to(s["q"].dtype)


def _plain_append(s):
    c, dev = s["case"], s["new"].device
    page, Hkv, D, S = c["page"], c["Hkv"], c["D"], c["S"]
    n = s["new_off"][1:] - s["new_off"][:-1]
    base = s["lens"] - n
    col = (base // page)[:, None] + torch.arange((c["nmax"] + page - 2) // page + 1, device=dev)[None, :]  # the pages a sequence may touch
    width = col.shape[1]
    at = col[:, :, None] * page + torch.arange(page, device=dev)
    fresh, old = (at >= base[:, None, None]) & (at < s["lens"][:, None, None]), at < base[:, None, None]
    rows = (s["new_off"][:-1] - base)[:, None, None] + at
    new = s["new"][rows.clamp_(0, s["new"].shape[0] - 1).long()].float()  # [S, width, page, 2, Hkv, D]
    ids = s["table"].gather(1, col.clamp(max=s["width"] - 1).long())
    ids = torch.where(fresh.any(-1), ids, s["n_pages"]).long()  # what is not touched goes to the spare page behind the last
    for i, x in enumerate("kv"):
        val, mask = new[:, :, :, i].transpose(2, 3), fresh[:, :, None, :, None]  # [S, width, Hkv, page, D]
        most = torch.where(mask, val.abs(), torch.zeros((), device=dev)).amax((-1, -2))
        m, ex = torch.frexp(most)
        need = torch.where(most > 0, ex - 9 + (m > 0.875).to(ex.dtype), torch.full_like(ex, -126)).clamp_(min=-126)
        e = torch.where(old.any(-1)[..., None], torch.maximum(torch.frexp(s[x + "_scale"][ids])[1] - 1, need), need)
        was = s[x][ids].float()
        grown = was * (s[x + "_scale"][ids] * torch.exp2(-e.float()))[..., None, None]
        codes = torch.where(mask, (val * torch.exp2(-e.float())[..., None, None]).clamp(-448, 448), torch.where(old[:, :, None, :, None], grown, was))
        s[x].view(torch.uint8)[ids] = codes.to(torch.float8_e4m3fn).view(torch.uint8)
        s[x + "_scale"][ids] = torch.exp2(e.float())
    return _whole(s)


def _plain_kv8(s):
    c, dev = s["case"], s["q"].device
    S, Q, T, Hkv, page = c["S"], c["nmax"], c["lmax"], c["Hkv"], c["page"]
    total, G = s["q"].shape[0], c["H"] // c["Hkv"]
    item, pos = _rows_of(s["q_off"], S, total)
    q = s["q"][_padded(s["q_off"], S, Q, total)].float().unflatten(2, (Hkv, G))
    ids = s["table"].long()
    k, v = ((s[x][ids].float() * s[x + "_scale"][ids][..., None, None]).transpose(2, 3).flatten(1, 2)[:, :T] for x in "kv")
    n = s["q_off"][1:] - s["q_off"][:-1]
    last = (s["lens"] - n)[:, None] + torch.arange(Q, device=dev)[None, :]
    at = torch.arange(T, device=dev)[None, None, :]
    return _attend(q, k, v, (at <= last[:, :, None]) & (at < s["lens"][:, None, None]), item, pos, 1 / math.sqrt(c["D"])).to(s["q"].dtype)


def _plain_select(s):
    c, dev = s["case"], s["cum"].device
    B, K, V = c["B"], c["K"], c["V"]
    x = s["logits"].view(B, K, V).double()  # sums over the vocabulary, and scores of different beams next to one another
    m = x.amax(-1, keepdim=True)
    lp = x - (m + torch.log(torch.exp(x - m).sum(-1, keepdim=True)))
    fin = s["finished"].bool()[..., None]
    eos = torch.arange(V, device=dev) == V - 1
    score = s["cum"].double()[..., None] + torch.where(fin, torch.where(eos, 0.0, float("-inf")).double(), lp)
    top, at = torch.sort(score.flatten(1), dim=1, descending=True, stable=True)
    at, parent = at[:, :K], at[:, :K] // V
    token = at - parent * V
    done = (token == V - 1) | s["finished"].bool().gather(1, parent)
    return {"score": top[:, :K].float(), "parent": parent.to(torch.int32), "token": token.to(torch.int32), "finished": done.to(torch.uint8)}


def _plain_rows(s):
    c = s["case"]
    B, K, live = c["B"], c["K"], c["live"]
    src = (torch.arange(B, device=s["parent"].device)[:, None] * K + s["parent"]).flatten().long()
    s["state"][:, :, :live] = s["state"][:, src, :live]
    return s["state"]


def _plain_pages(s):
    c, dev = s["case"], s["parent"].device
    B, K, page = c["B"], c["K"], c["page"]
    src = (torch.arange(B, device=dev)[:, None] * K + s["parent"]).flatten().long()
    full = (s["lens"] // page)[:, None]
    col = torch.arange(s["width"], device=dev)[None, :]
    mine = s["table"].gather(1, full.clamp(max=s["width"] - 1).long())[:, 0].long()  # each sequence's page that is being filled
    part = s["lens"] % page
    live = (torch.arange(page, device=dev)[None, :] < part[:, None])[:, None, :, None]
    for x in "kv":
        codes = s[x].view(torch.uint8)
        codes[mine] = torch.where(live, codes[mine[src]], codes[mine])
        s[x + "_scale"][mine] = torch.where((part > 0)[:, None], s[x + "_scale"][mine[src]], s[x + "_scale"][mine])
    s["table"].copy_(torch.where(col < full, s["table"][src], s["table"]))
    return _whole(s, "table")


# ---------------------------------------------------------------- the library's calls


def _pkc():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "parakeet.cpp_b200", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    import pkc
    return pkc


def _own_cache(s, pkc, **more):
    c = s["case"]
    if "cache" not in s:
        s["cache"] = pkc.KV8Cache(k=s["k"].data_ptr(), v=s["v"].data_ptr(), k_scale=s["k_scale"].data_ptr(), v_scale=s["v_scale"].data_ptr(), table=s["table"].data_ptr(),
                                  n_pages=s["n_pages"], page=c["page"], n_kv_heads=c["Hkv"], head_dim=c["D"], table_ld=s["width"])
        s["err"] = torch.zeros(1, dtype=torch.int32, device=s["k"].device)
    return s["cache"]


def _workspace(s, bytes_, dev):
    if "work" not in s:
        s["work"] = torch.empty(max(16, bytes_), dtype=torch.uint8, device=dev)
    return s["work"]


def _own_run(s):
    pkc, c, op = _pkc(), s["case"], s["case"]["op"]
    st = torch.cuda.current_stream().cuda_stream
    if op == "cross":
        H, Hkv, D = c["H"], c["Hkv"], c["D"]
        w = s.get("work")
        if w is None:
            w = _workspace(s, pkc.cross_attention_workspace(c["B"], c["qmax"], c["tmax"], H, Hkv, D), s["q"].device)
        pkc.cross_attention(s["q"].data_ptr(), s["kv"].data_ptr(), s["kv"][:, 1].data_ptr(), s["q_off"].data_ptr(), s["kv_off"].data_ptr(), s["kv_len"].data_ptr(), c["B"], H, Hkv, D,
                            q_rows=s["q"].shape[0], kv_rows=s["kv"].shape[0], max_q=c["qmax"], max_kv=c["tmax"], ldk=2 * Hkv * D, ldv=2 * Hkv * D, bf16=c["dtype"] == "bf16",
                            out=s["out"].data_ptr(), workspace=w.data_ptr(), workspace_bytes=w.numel(), stream=st)
        return s["out"]
    if op == "append":
        Hkv, D = c["Hkv"], c["D"]
        pkc.kv8_append(_own_cache(s, pkc), s["new"].data_ptr(), s["new"][:, 1].data_ptr(), s["new_off"].data_ptr(), s["lens"].data_ptr(), c["S"], rows=s["new"].shape[0], max_new=c["nmax"],
                       ldk=2 * Hkv * D, ldv=2 * Hkv * D, bf16=c["dtype"] == "bf16", err=s["err"].data_ptr(), stream=st)
        return _whole(s)
    if op == "kv8":
        cache, w = _own_cache(s, pkc), s.get("work")
        if w is None:
            w = _workspace(s, pkc.kv8_attention_workspace(cache, c["S"], c["nmax"], c["lmax"], c["H"]), s["q"].device)
        pkc.kv8_attention(cache, s["q"].data_ptr(), s["q_off"].data_ptr(), s["lens"].data_ptr(), c["S"], c["H"], q_rows=s["q"].shape[0], max_q=c["nmax"], max_len=c["lmax"],
                          bf16=c["dtype"] == "bf16", out=s["out"].data_ptr(), workspace=w.data_ptr(), workspace_bytes=w.numel(), err=s["err"].data_ptr(), stream=st)
        return s["out"]
    if op == "select":
        pkc.beam_select(s["logits"].data_ptr(), s["cum"].data_ptr(), s["finished"].data_ptr(), c["B"], c["K"], c["V"], eos=c["V"] - 1, dtype=c["dtype"], score=s["score"].data_ptr(),
                        parent=s["parent"].data_ptr(), token=s["token"].data_ptr(), finished_out=s["done"].data_ptr(), stream=st)
        return {"score": s["score"], "parent": s["parent"], "token": s["token"], "finished": s["done"]}
    if op == "rows":
        x = s["state"]
        size = x.element_size() * c["unit"]
        pkc.beam_reorder(x.data_ptr(), s["parent"].data_ptr(), c["B"], c["K"], row_bytes=c["live"] * size, row_stride=c["cap"] * size, n_outer=c["outer"],
                         outer_stride=c["B"] * c["K"] * c["cap"] * size, stream=st)
        return x
    pkc.kv8_reorder(_own_cache(s, pkc), s["parent"].data_ptr(), s["lens"].data_ptr(), c["B"], c["K"], err=s["err"].data_ptr(), stream=st)
    return _whole(s, "table")


def run(state):
    if own:
        return _own_run(state)
    plain = {"cross": _plain_cross, "append": _plain_append, "kv8": _plain_kv8, "select": _plain_select, "rows": _plain_rows, "pages": _plain_pages}
    return plain[state["case"]["op"]](state)


# ---------------------------------------------------------------- work and exact values


def work(case):
    c, op = case, case["op"]
    a, b = _sizes(c)
    if op == "cross":
        row = 2 * c["D"]
        return {"bytes": 2 * sum(a) * c["H"] * row + 2 * sum(t for t in b) * c["Hkv"] * row, "flops": 4.0 * c["D"] * c["H"] * sum(x * t for x, t in zip(a, b))}
    if op == "append":
        # new rows in, their codes and the scales of their pages out
        return {"bytes": sum(a) * 2 * c["Hkv"] * c["D"] * 3 + sum(-(-n // c["page"]) for n in a) * 2 * c["Hkv"] * 8, "flops": 4 * sum(a) * 2 * c["Hkv"] * c["D"]}
    if op == "kv8":
        seen = sum(n * t - n * (n - 1) / 2 for n, t in zip(a, b))
        return {"bytes": 4 * sum(a) * c["H"] * c["D"] + 2 * c["Hkv"] * sum(t * c["D"] + 4 * -(-t // c["page"]) for t in b), "flops": 4.0 * c["D"] * c["H"] * seen}
    if op == "select":
        return {"bytes": c["B"] * c["K"] * c["V"] * (4 if c["dtype"] == "f32" else 2) + c["B"] * c["K"] * 18, "flops": 4.0 * c["B"] * c["K"] * c["V"]}
    # every row may have to move: a share of them keeps its place (its parent is itself), 0.4 + 0.6 / K of them on average
    moved = 0.6 * (1 - 1 / c["K"])
    if op == "rows":
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": 2 * moved * c["outer"] * c["B"] * c["K"] * c["live"] * c["unit"] * size, "flops": 0}
    return {"bytes": 2 * moved * c["K"] * sum(2 * c["Hkv"] * ((t % c["page"]) * c["D"] + 4) + 4 * (t // c["page"]) for t in b), "flops": 0}


def _softmax_rows(q, k, v, first, scale):
    """q [n, G, D], k / v [t, D] in 64 bits; row i sees its first `first + i` keys, or all where first is None."""
    s = (q.reshape(-1, q.shape[-1]) @ k.T).view(q.shape[0], q.shape[1], -1) * scale
    if first is not None:
        sees = first + torch.arange(q.shape[0], device=q.device)
        s = s.masked_fill(torch.arange(k.shape[0], device=q.device)[None, None, :] >= sees[:, None, None], float("-inf"))
    return (torch.softmax(s, -1).view(-1, k.shape[0]) @ v).view(q.shape)


def _to_e4m3(x):
    """The nearest value of 4 exponent and 3 mantissa bits, ties to even, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_append(s, a, b):
    c, page = s["case"], s["case"]["page"]
    new, table, r0, res = s["new"].double(), s["table"].tolist(), 0, {}
    codes = {x: s[x][: s["n_pages"]].double() for x in "kv"}
    scale = {x: s[x + "_scale"][: s["n_pages"]].double() for x in "kv"}
    jobs = []
    for i, (n, length) in enumerate(zip(a, b)):
        for p in range((length - n) // page, -(-length // page) if n else 0):
            lo, hi = max(length - n, p * page), min(length, (p + 1) * page)
            jobs.append((table[i][p], lo - p * page, hi - p * page, r0 + lo - (length - n)))
        r0 += n
    if jobs:
        j = torch.tensor(jobs, device=new.device)
        at = torch.arange(page, device=new.device)[None, :]
        fresh, old = ((at >= j[:, 1:2]) & (at < j[:, 2:3]))[:, None, :, None], (at < j[:, 1:2])[:, None, :, None]
        rows = (j[:, 3:4] + at - j[:, 1:2]).clamp(0, new.shape[0] - 1)
        for i, x in enumerate("kv"):
            val = new[rows][:, :, i].transpose(1, 2)
            most = torch.where(fresh, val.abs(), 0.0).amax((-1, -2))
            need = torch.ceil(torch.log2(most.clamp(min=1e-300) / 448)).clamp(min=-126)
            need = need - (most <= 448 * torch.exp2(need - 1)).double() * (need > -126)
            need = need + (most > 448 * torch.exp2(need)).double()
            was = scale[x][j[:, 0]]
            now = torch.where(old.any(2)[..., 0], torch.maximum(was, torch.exp2(need)), torch.exp2(need))
            ratio, now4 = (was / now)[..., None, None], now[..., None, None]
            was4 = codes[x][j[:, 0]]
            codes[x][j[:, 0]] = torch.where(fresh, _to_e4m3(val / now4), torch.where(old, _to_e4m3(was4 * ratio), was4))
            scale[x][j[:, 0]] = now
    for x in "kv":
        res[x], res[x + "_scale"] = codes[x], scale[x]
    return res


def exact(case, seed):
    c, op = case, case["op"]
    s = prepare(case, seed)
    a, b = _sizes(c)
    if op == "append":
        return _exact_append(s, a, b)
    if op in ("cross", "kv8"):
        G, out, r0, t0 = c["H"] // c["Hkv"], [], 0, 0
        for i, (n, t) in enumerate(zip(a, b)):
            q = s["q"][r0:r0 + n].double()
            if op == "cross":
                k, v = s["kv"][t0:t0 + t].double().unbind(1)
            else:
                ids = s["table"][i, : -(-t // c["page"])].long()
                k, v = ((s[x][ids].double() * s[x + "_scale"][ids].double()[..., None, None]).transpose(1, 2).flatten(0, 1)[:t] for x in "kv")
            o = torch.zeros_like(q)
            for h in range(c["Hkv"] if t else 0):
                o[:, h * G:(h + 1) * G] = _softmax_rows(q[:, h * G:(h + 1) * G], k[:, h], v[:, h], t - n + 1 if op == "kv8" else None, 1 / math.sqrt(c["D"]))
            out.append(o)
            r0, t0 = r0 + n, t0 + t
        return torch.cat(out)
    if op == "select":
        B, K, V = c["B"], c["K"], c["V"]
        lp = torch.log_softmax(s["logits"].double().view(B, K, V), -1)
        lp = torch.where(s["finished"].bool()[..., None], float("-inf"), lp)
        lp[..., V - 1] = torch.where(s["finished"].bool(), 0.0, lp[..., V - 1])
        best = (lp + s["cum"].double()[..., None]).flatten(1).topk(K, dim=1)[0]
        return {"score": best, "parent": None, "token": None, "finished": None}
    return None  # the reordering moves bits
