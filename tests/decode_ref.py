"""Plain 64-bit restatements of the attention decoder's operators and the
error bounds that the tests hold the kernels to."""
import math

import torch


def need_exp(most):
    """The smallest integer e >= -126 with most <= 448 * 2^e."""
    if most <= 0:
        return -126
    e = math.ceil(math.log2(most / 448.0))
    while most > 448.0 * 2.0 ** e:
        e += 1
    while most <= 448.0 * 2.0 ** (e - 1):
        e -= 1
    return max(e, -126)


def to_e4m3(x):
    """Nearest e4m3 value of a float64 tensor (ties to even, saturating)."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


class RefCache:
    """A paged cache in float64: codes as the values of e4m3, scales as
    exponents, updated one page and head at a time by the definition."""

    def __init__(self, n_pages, Hkv, page, D):
        self.page, self.Hkv, self.D = page, Hkv, D
        self.code = torch.zeros(2, n_pages, Hkv, page, D, dtype=torch.float64)
        self.exp = torch.full((2, n_pages, Hkv), -126)

    def append(self, table, new, length):
        """new [n, 2, Hkv, D] float64 become the last n of `length` tokens of
        the sequence whose pages are `table`."""
        n = new.shape[0]
        base = length - n
        for p in range(base // self.page, -(-length // self.page) if n else 0):
            lo, hi = max(base, p * self.page), min(length, (p + 1) * self.page)
            at, used = int(table[p]), lo - p * self.page
            for x in range(2):
                for h in range(self.Hkv):
                    v = new[lo - base:hi - base, x, h]
                    v = torch.where(torch.isnan(v), torch.zeros_like(v), v)
                    fin = v[torch.isfinite(v)].abs()
                    e = need_exp(float(fin.max()) if fin.numel() else 0.0)
                    if used:
                        old = int(self.exp[x, at, h])
                        e = max(e, old)
                        self.code[x, at, h, :used] = to_e4m3(self.code[x, at, h, :used] * 2.0 ** (old - e))
                    self.exp[x, at, h] = e
                    self.code[x, at, h, used:used + hi - lo] = to_e4m3(v * 2.0 ** -e)

    def dense(self, table, length):
        """(k, v) [length, Hkv, D] float64 of a sequence."""
        ids = torch.as_tensor([int(t) for t in table[: -(-length // self.page)]], dtype=torch.long)
        out = []
        for x in range(2):
            val = self.code[x, ids] * torch.exp2(self.exp[x, ids].double())[..., None, None]
            out.append(val.transpose(1, 2).reshape(-1, self.Hkv, self.D)[:length])
        return out


def attention(q, k, v, scale, causal):
    """q [n, H, D], k / v [t, Hkv, D] float64. Returns (o, A, S): the output,
    sum_j p_ij |v_j| and the largest sum_d |q_d k_d| * scale of each row."""
    n, H, D = q.shape
    t, G = k.shape[0], H // k.shape[1]
    if t == 0:
        z = torch.zeros_like(q)
        return z, z.clone(), torch.zeros(n, H, 1, dtype=q.dtype, device=q.device)
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = torch.einsum("nhd,thd->hnt", q, k) * scale
    mag = torch.einsum("nhd,thd->hnt", q.abs(), k.abs()).amax(-1) * abs(scale)
    if causal:
        sees = t - n + 1 + torch.arange(n, device=q.device)
        s = s.masked_fill(torch.arange(t, device=q.device)[None, None, :] >= sees[None, :, None], float("-inf"))
    p = torch.softmax(s, -1)
    o, A = (torch.einsum("hnt,thd->nhd", p, x) for x in (v, v.abs()))
    return o, A, mag.T[..., None]


def attention_tolerance(o, A, S, v_max, t, D, out_dtype, p_dtype):
    """How far a kernel's output may be from o, element by element.

    Scores: sums of D products in f32, at most (D + 8) 2^-24 of the sum of
    their magnitudes off, and the exponent function 2^-21; such an error d of
    every score changes each weight by a factor within exp(+-2 d). Each
    probability is then rounded to p_dtype: half a step of it, relative, or,
    in f16, 2^-25 where it is below the normal range (probabilities are at most
    1 and their sum at least 1). The sums in f32 over t keys: (t + 8) 2^-24
    where parts are joined in any order. Last the rounding of the output."""
    eps = torch.finfo(p_dtype).eps / 2
    d = (D + 8) * 2.0 ** -24 * S + 2.0 ** -21
    tol = A * (torch.expm1(2 * d) + eps + (min(t, 4096) + 8) * 2.0 ** -23)
    if p_dtype == torch.float16:
        tol = tol + t * 2.0 ** -25 * v_max
    return tol * 1.01 + o.abs() * (torch.finfo(out_dtype).eps / 2) * 1.01 + 2.0 ** -24


def beam_select(logits, cum, finished, eos):
    """logits [B, K, V], cum [B, K], finished [B, K] bool -> (score f64, parent, token, finished)."""
    B, K, V = logits.shape
    x = logits.double()
    lse = torch.logsumexp(x, -1, keepdim=True)
    lp = torch.where(torch.isfinite(lse), x - lse, torch.full_like(x, float("-inf")))
    only = torch.full((V,), float("-inf"), dtype=torch.float64, device=x.device)
    only[eos] = 0.0
    lp = torch.where(finished[..., None], only, lp)
    sc = cum.double()[..., None] + lp
    sc = torch.where(torch.isnan(sc), torch.full_like(sc, float("-inf")), sc).flatten(1)
    top, at = torch.sort(sc, dim=1, descending=True, stable=True)
    top, at = top[:, :K], at[:, :K]
    parent, token = at // V, at % V
    return top, parent, token, (token == eos) | finished.gather(1, parent)
